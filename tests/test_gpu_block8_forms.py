"""The layer half over 8-bit rows (senmoe.block8): that a step's gradients are
the same bits every time, and what it refuses."""
import pytest
from test_gpu_block8 import _block

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


def test_gradients_repeat(senmoe, torch):
    """Rows of eight experts meet in a token's gradient, in one order: equal bits, and no step of it that adds by
    atomics, whose order shows in few of the rounded results."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        names = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.add(func.overloadpacket.__name__)
            return func(*args, **(kwargs or {}))
    block, x, r = _block(senmoe, torch, 1031, 512, 96, 32, 8, 64)
    out, saved = block.forward(x, residual=r, train=True)
    with Seen() as seen:
        dx, grads = block.backward(out, saved)
    assert "index" in seen.names  # (it does see them)
    assert not {n for n in seen.names if "index_add" in n or "scatter_add" in n or "index_put" in n or "bincount" in n}
    for _ in range(20):
        again, g = block.backward(out, saved)
        assert torch.equal(again, dx)
        assert all(torch.equal(g[k], v) for k, v in grads.items())


def test_block_refuses(senmoe, torch):
    """Rows and router weights of another type, which the router would read as bf16, and of other dimensions."""
    block, x, r = _block(senmoe, torch, 6, 256, 96, 8, 2, 0)
    for dtype in (torch.float16, torch.float32):
        with pytest.raises(TypeError):
            block.forward(x.to(dtype), residual=r.to(dtype))
    for bad in (x.view(2, 3, 256), x[0], x[:, :128]):
        with pytest.raises(senmoe.SenMoeError):
            block.forward(bad)
    block.w.router = block.w.router.half()
    with pytest.raises(TypeError):
        block.forward(x, residual=r)
    torch.cuda.synchronize()


@pytest.mark.parametrize("T,shared", [(1, 0), (37, 64), (300, 128)])
def test_inference_gives_what_training_does(senmoe, torch, T, shared):
    """The products choose their kernels by sizes alone, whether or not pre-activations are kept."""
    block, x, r = _block(senmoe, torch, T, 512, 96, 16, 4, shared)
    out, _ = block.forward(x, residual=r, train=True)
    assert torch.equal(block.forward(x, residual=r), out)
