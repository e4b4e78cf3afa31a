"""CPU tests of the 16-bit linear products' boundary: struct layouts, the C
checks that come before any CUDA call, and the Python checks."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


@pytest.fixture(scope="module")
def senmoe():
    import build as b
    b.build()
    import senmoe as s
    return s


def test_struct_layouts(senmoe):
    prog = "#include <stdio.h>\n#include <stddef.h>\n#include \"senmoe.h\"\nint main(void) {\n"
    want = []
    for t in (senmoe.SenMoeLinear, senmoe.SenMoeLinearGrad):
        prog += f'printf("%zu ", sizeof({t.__name__}));\n'
        want.append(C.sizeof(t))
        for name, _ in t._fields_:
            prog += f'printf("%zu ", offsetof({t.__name__}, {name}));\n'
            want.append(getattr(t, name).offset)
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write(prog + "return 0; }\n")
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == want


def _product(senmoe, **kw):
    q = senmoe.SenMoeLinear(0, 0, 1, 0, 4, 64, 32, 0x10000, 64, 0x20000, 64, 64 * 32, None, None, None, 0, 0x30000, 32,
                            None, 0)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize("kw,status,word", [
    (dict(dtype=2), 5, "dtype"), (dict(epilogue=7), 5, "epilogue"), (dict(epilogue=-1), 5, "epilogue"),
    (dict(path=9), 1, "path"), (dict(num_groups=0), 1, "num_groups"), (dict(num_groups=3), 1, "without offsets"),
    (dict(num_groups=1025, offsets=0x40000), 5, "1024"), (dict(offsets=0x40002), 1, "offsets"),
    (dict(rows=-1), 1, "rows"), (dict(rows=1 << 31), 1, "rows"), (dict(in_features=0), 1, "in_features"),
    (dict(out_features=0), 1, "out_features"), (dict(x=None), 1, "x is NULL"), (dict(x=0x10001), 1, "aligned"),
    (dict(x_stride=63), 1, "stride"), (dict(weight=None), 1, "weight"), (dict(weight_stride=10), 1, "stride"),
    (dict(num_groups=2, offsets=0x40000, weight_group_stride=100), 1, "group stride"), (dict(y=None), 1, "y is NULL"),
    (dict(y_stride=31), 1, "stride"), (dict(residual=0x50000, residual_stride=3), 1, "residual"),
    (dict(preact=0x50000, preact_stride=3), 1, "preact"), (dict(epilogue=5, preact=0x50000, preact_stride=32), 1, "preact"),
    (dict(bias=0x50001), 1, "bias"),
])
def test_linear_rejects(senmoe, kw, status, word):
    L = senmoe.lib()
    assert L.senmoe_linear(C.byref(_product(senmoe, **kw)), None) == status
    assert word in L.senmoe_last_error().decode()


def test_linear_nothing_to_do(senmoe):
    assert senmoe.lib().senmoe_linear(C.byref(_product(senmoe, rows=0, x=None, y=None)), None) == 0
    assert senmoe.lib().senmoe_linear(None, None) == 1


def _grad(senmoe, **kw):
    g = senmoe.SenMoeLinearGrad(0, 2, 1, 0, 4, 64, 32, 0x10000, 32, 0x20000, 64, 0x30000, 64, 64 * 32, None, 0x40000,
                                32, 0x50000, 64, 0x60000, 64, 64 * 32, 0x70000, 0x80000, 1 << 20)
    for k, v in kw.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize("kw,word", [
    (dict(dy=None), "dy is NULL"), (dict(dy_stride=8), "stride"), (dict(preact=None), "preact is NULL"),
    (dict(x=None), "x is NULL"), (dict(weight=None), "weight is NULL"), (dict(dx_stride=2), "dx"),
    (dict(dweight_stride=2), "dweight"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=16), "workspace"),
    (dict(workspace=0x80008), "aligned"), (dict(dbias=0x70001), "dbias"),
    (dict(num_groups=2, offsets=0x90000, dweight_group_stride=64), "dweight group stride"),
])
def test_linear_backward_rejects(senmoe, kw, word):
    L = senmoe.lib()
    assert L.senmoe_linear_backward(C.byref(_grad(senmoe, **kw)), None) == 1
    assert word in L.senmoe_last_error().decode()


def test_backward_workspace(senmoe):
    L = senmoe.lib()
    size = lambda **kw: L.senmoe_linear_backward_workspace(C.byref(_grad(senmoe, **kw)))  # noqa: E731
    assert size(epilogue=0) == 0
    assert size() == 4 * 32 * 2                         # dz
    assert size(epilogue=5) == 4 * 64 * 2               # dz of gate and up
    assert size(out_features=33, dy_stride=33) == 4 * 40 * 2  # its rows in steps of 16 bytes
    assert size(rows=0) == 0
    assert size(dtype=3) == -5 and L.senmoe_last_error()


def test_python_checks(senmoe):
    import torch
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError):  # no CPU path
        senmoe.linear(x, w)
    with pytest.raises(TypeError):
        senmoe.linear(x.float(), w.float())
    with pytest.raises(senmoe.SenMoeError, match="activation"):
        senmoe.linear(x, w, activation="tanh")
    with pytest.raises(senmoe.SenMoeError, match="weight must be"):
        senmoe.linear(x, w[None])
    with pytest.raises(senmoe.SenMoeError, match="experts"):
        senmoe.grouped_linear(x, w, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="int32"):
        senmoe.grouped_linear(x, w[None], torch.zeros(2, dtype=torch.int64))
    with pytest.raises(senmoe.SenMoeError, match="offsets"):
        senmoe.grouped_linear(x, w[None], torch.zeros(3, dtype=torch.int32))
    with pytest.raises(senmoe.SenMoeError, match="rows"):
        senmoe.grouped_linear(x[None], w[None], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError):
        senmoe.linear_backward(torch.zeros(4, 32, dtype=torch.bfloat16), x, w)
