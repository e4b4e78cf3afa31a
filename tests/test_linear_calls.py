"""CPU tests of what the linear products' calls do before anything is launched."""
import contextlib

import pytest


@pytest.fixture(scope="module")
def senmoe():
    import build as b
    b.build()
    import senmoe as s
    return s


class _Copied(Exception):
    pass


class _StridedOffsets:
    """Stands for int32 offsets that are not contiguous: says where they are copied."""

    def __init__(self, torch, inside):
        self.dtype, self.device, self.shape, self.inside = torch.int32, "cpu", (2,), inside

    def dim(self):
        return 1

    def get_device(self):
        return -1

    def contiguous(self):
        raise _Copied(list(self.inside))


@pytest.mark.parametrize("backward", [False, True])
def test_offsets_are_copied_on_the_launch_stream(senmoe, monkeypatch, backward):
    import torch
    from senmoe import products
    inside = []

    @contextlib.contextmanager
    def stream(s):
        inside.append(s)
        yield
        inside.pop()
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(products, "_operands", lambda *t: (0, -1))
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(1, 32, 64, dtype=torch.bfloat16)
    off = _StridedOffsets(torch, inside)
    with pytest.raises(_Copied) as e:
        if backward:
            senmoe.grouped_linear_backward(torch.zeros(4, 32, dtype=torch.bfloat16), x, w, off, stream="launch")
        else:
            senmoe.grouped_linear(x, w, off, stream="launch")
    assert e.value.args[0] == ["launch"]


def test_import_without_a_cuda_build_of_torch():
    """The loader and the synthetic weights are used on hosts whose torch has no CUDA build."""
    import os
    import subprocess
    import sys
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "sen-mlx_b200")
    prog = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]: delattr(torch._C, n)\n"
            "import senmoe, senmoe.loader, senmoe.synth\n")
    subprocess.run([sys.executable, "-c", prog], check=True, cwd=root, timeout=300)


def _bf16(*shape):
    import torch
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("call,word", [
    (lambda m: m.linear(_bf16(4, 0), _bf16(8, 0)), "in_features=0"),
    (lambda m: m.linear(_bf16(4, 8), _bf16(0, 8), activation="swiglu"), "out_features=0"),
    (lambda m: m.linear_backward(_bf16(4, 8), _bf16(4, 0), _bf16(8, 0)), "in_features=0"),
    (lambda m: m.linear_backward(_bf16(2, 2, 0), _bf16(2, 2, 8), _bf16(0, 8)), "out_features=0"),
    (lambda m: m.linear(_bf16(4, 8), _bf16(1, 8), bias=_bf16(())), "bias"),
    (lambda m: m.linear(_bf16(2, 3, 8), _bf16(8, 8), out=_bf16(3, 2, 8).transpose(0, 1)), "out"),
])
def test_bad_shapes_are_refused_in_the_packages_manner(senmoe, monkeypatch, call, word):
    from senmoe import products
    monkeypatch.setattr(products, "_operands", lambda *t: (0, -1))
    with pytest.raises(senmoe.SenMoeError, match=word) as e:
        call(senmoe)
    assert e.value.status == senmoe.ERR_BAD_ARG


def test_finetuning_stops_before_a_failed_step_is_taken(senmoe, monkeypatch):
    """A wait that ran out leaves garbage gradients: no weight takes them."""
    import os
    import sys
    import types

    import torch
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
    import moe_finetune
    names = ("gate_up", "down", "shared_gate_up", "shared_down")
    w = types.SimpleNamespace(**{n: torch.ones(2, 2, dtype=torch.bfloat16) for n in names})
    x = torch.ones(3, 2, dtype=torch.bfloat16)
    block = types.SimpleNamespace(w=w, forward=lambda x, train=False: (2 * x, None) if train else x,
                                  backward=lambda dh, saved: (dh, {n: torch.ones(2, 2) for n in names}))

    def ran_out(stream=None):
        raise senmoe.SenMoeError(senmoe.ERR_TIMEOUT, "a wait ran out")
    monkeypatch.setattr(senmoe, "linear_check", ran_out)
    with pytest.raises(senmoe.SenMoeError):
        moe_finetune.train(block, block, x, steps=2, lr=0.5)
    assert all((getattr(w, n) == 1).all() for n in names)
