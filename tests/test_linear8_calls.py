"""CPU tests of what the calls on 8-bit rows and the norm refuse before
anything is launched, and of their structs' layout."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
BAD, UNSUPPORTED, OK = 1, 5, 0
P = 0x10000  # never read: every call here is refused, or has no rows


@pytest.fixture(scope="module")
def senmoe():
    import build as b
    b.build()
    import senmoe as s
    return s


def test_struct_layouts(senmoe, tmp_path):
    names = ["SenMoeNorm", "SenMoeNormGrad", "SenMoeQuantize8", "SenMoeLinear8"]
    lines = "\n".join(f'printf("%zu", sizeof({n}));' + "".join(
        f'printf(" %zu", offsetof({n}, {f}));' for f, _ in getattr(senmoe, n)._fields_) + 'printf("\\n");' for n in names)
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "senmoe.h"\nint main(void) {{ {lines} return 0; }}')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.strip().split("\n")
    for n, line in zip(names, out):
        s = getattr(senmoe, n)
        assert [int(v) for v in line.split()] == [C.sizeof(s), *(getattr(s, f).offset for f, _ in s._fields_)], n


def test_packed_arguments_match_the_structs(senmoe):
    """The calls pack their argument structs themselves."""
    from senmoe import norm, products8
    for pack, s in ((norm._pack_norm, senmoe.SenMoeNorm), (norm._pack_grad, senmoe.SenMoeNormGrad),
                    (products8._pack_quantize, senmoe.SenMoeQuantize8), (products8._pack_linear8, senmoe.SenMoeLinear8)):
        v = [float(i) if t is C.c_float else i for i, (_, t) in enumerate(s._fields_)]
        raw = pack(*v)
        got = s.from_buffer_copy(raw.ljust(C.sizeof(s), b"\0"))
        assert len(raw) <= C.sizeof(s) and [getattr(got, f) or 0 for f, _ in s._fields_] == v


def _fill(s, **kw):
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _linear8(senmoe, **kw):
    base = dict(dtype=0, epilogue=0, num_groups=1, path=0, rows=4, in_features=64, out_features=32, x=P, x_stride=64,
                x_scales=P, x_scales_stride=2, weight=P, weight_stride=64, weight_group_stride=2048, weight_scales=P,
                weight_scales_stride=2, weight_scales_group_stride=64, y=P, y_stride=32)
    return senmoe.lib().senmoe_linear8(C.byref(_fill(senmoe.SenMoeLinear8(), **{**base, **kw})), None)


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 2}, UNSUPPORTED), ({"epilogue": 7}, UNSUPPORTED), ({"path": 7}, BAD), ({"path": 1}, UNSUPPORTED),
    ({"num_groups": 0}, BAD), ({"num_groups": 2}, BAD), ({"num_groups": 1025, "offsets": P}, UNSUPPORTED),
    ({"offsets": P + 1}, BAD), ({"rows": -1}, BAD), ({"rows": 1 << 31}, BAD), ({"in_features": 0}, BAD),
    ({"in_features": 48}, UNSUPPORTED), ({"out_features": 0}, BAD), ({"y": None}, BAD), ({"y_codes": P}, BAD),
    ({"y": None, "y_codes": P, "y_codes_stride": 32}, BAD),
    ({"y": None, "y_codes": P, "y_codes_stride": 48, "y_scales": P, "y_scales_stride": 1, "out_features": 40}, UNSUPPORTED),
    ({"y": None, "y_codes": P + 8, "y_codes_stride": 32, "y_scales": P, "y_scales_stride": 1}, UNSUPPORTED),
    ({"x": None}, BAD), ({"x_scales": None}, BAD), ({"x": P + 8}, UNSUPPORTED), ({"x_stride": 72}, UNSUPPORTED),
    ({"x_stride": 32}, BAD), ({"x_scales_stride": 1}, BAD), ({"weight": None}, BAD), ({"weight": P + 4}, UNSUPPORTED),
    ({"weight_stride": 100}, UNSUPPORTED), ({"weight_scales_stride": 1}, BAD),
    ({"num_groups": 2, "offsets": P, "weight_group_stride": 1024}, BAD),
    ({"num_groups": 2, "offsets": P, "weight_group_stride": 2056}, UNSUPPORTED),
    ({"num_groups": 2, "offsets": P, "weight_scales_group_stride": 32}, BAD),
    ({"y": P + 1}, BAD), ({"y_stride": 16}, BAD), ({"residual": P, "residual_stride": 16}, BAD),
    ({"preact": P, "preact_stride": 16}, BAD), ({"bias": P + 1}, BAD),
    ({"rows": (1 << 31) - 1024, "out_features": 1 << 20}, UNSUPPORTED),
    ({"path": 3, "rows": 600000}, UNSUPPORTED),
])
def test_linear8_refuses(senmoe, kw, status):
    assert _linear8(senmoe, **kw) == status, senmoe.lib().senmoe_last_error()
    assert senmoe.lib().senmoe_last_error()


def test_calls_without_rows_do_nothing(senmoe):
    L = senmoe.lib()
    assert _linear8(senmoe, rows=0, x=None, weight=None, y=None) == OK
    q = _fill(senmoe.SenMoeQuantize8(), rows=0, n=64)
    assert L.senmoe_quantize8(C.byref(q), None) == OK
    n = _fill(senmoe.SenMoeNorm(), rows=0, hidden=64, eps=1e-6)
    assert L.senmoe_rms_norm(C.byref(n), None) == OK
    g = _fill(senmoe.SenMoeNormGrad(), rows=0, hidden=64, eps=1e-6)
    assert L.senmoe_rms_norm_backward_workspace(C.byref(g)) == 0 and L.senmoe_rms_norm_backward(C.byref(g), None) == OK
    for f in (L.senmoe_linear8, L.senmoe_quantize8, L.senmoe_rms_norm, L.senmoe_rms_norm_backward):
        assert f(None, None) == BAD
    assert L.senmoe_rms_norm_backward_workspace(None) == -BAD


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 3}, UNSUPPORTED), ({"epilogue": -1}, UNSUPPORTED), ({"rows": -2}, BAD), ({"n": 0}, BAD), ({"n": 40}, UNSUPPORTED),
    ({"x": None}, BAD), ({"x": P + 1}, BAD), ({"x_stride": 32}, BAD), ({"epilogue": 2}, BAD),
    ({"epilogue": 5, "preact": P, "preact_stride": 64}, BAD), ({"codes": None}, BAD), ({"codes": P + 2}, UNSUPPORTED),
    ({"codes_stride": 70}, UNSUPPORTED), ({"scales": None}, BAD), ({"scales_stride": 1}, BAD),
])
def test_quantize8_refuses(senmoe, kw, status):
    base = dict(dtype=1, epilogue=0, rows=4, n=64, x=P, x_stride=64, codes=P, codes_stride=64, scales=P, scales_stride=2)
    q = _fill(senmoe.SenMoeQuantize8(), **{**base, **kw})
    assert senmoe.lib().senmoe_quantize8(C.byref(q), None) == status


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 2}, UNSUPPORTED), ({"weight_fp32": 2}, BAD), ({"unit_offset": -1}, BAD), ({"eps": -1.0}, BAD),
    ({"eps": float("nan")}, BAD), ({"rows": -1}, BAD), ({"hidden": 0}, BAD), ({"hidden": 1 << 25}, BAD), ({"weight": None}, BAD),
    ({"weight": P + 2, "weight_fp32": 1}, BAD), ({"x": None}, BAD), ({"x_stride": 10}, BAD), ({"y": None}, BAD),
    ({"residual": P + 1, "residual_stride": 64}, BAD), ({"y": None, "h": P, "h_stride": 64}, BAD),
    ({"codes": P, "codes_stride": 64}, BAD), ({"codes": P, "codes_stride": 64, "scales": P, "scales_stride": 1}, BAD),
    ({"codes": P, "codes_stride": 64, "scales": P, "scales_stride": 2, "hidden": 40}, UNSUPPORTED),
])
def test_rms_norm_refuses(senmoe, kw, status):
    base = dict(dtype=0, eps=1e-6, rows=4, hidden=64, x=P, x_stride=64, weight=P, y=P, y_stride=64)
    n = _fill(senmoe.SenMoeNorm(), **{**base, **kw})
    assert senmoe.lib().senmoe_rms_norm(C.byref(n), None) == status


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 2}, UNSUPPORTED), ({"hidden": 0}, BAD), ({"weight": None}, BAD), ({"dy": None}, BAD), ({"h": P + 1}, BAD),
    ({"dh": P, "dh_stride": 3}, BAD), ({"dx": P + 1, "dx_stride": 64}, BAD), ({"dweight": P + 1}, BAD), ({"workspace": None}, BAD),
    ({"workspace_bytes": 4}, BAD), ({"workspace": P + 8}, BAD),
])
def test_rms_norm_backward_refuses(senmoe, kw, status):
    base = dict(dtype=0, eps=1e-6, rows=4, hidden=64, dy=P, dy_stride=64, h=P, h_stride=64, weight=P, dweight=P, workspace=P,
                workspace_bytes=1 << 20)
    g = _fill(senmoe.SenMoeNormGrad(), **{**base, **kw})
    assert senmoe.lib().senmoe_rms_norm_backward(C.byref(g), None) == status


def test_python_refusals(senmoe):
    """Wrong types, shapes and devices raise as the linear products' calls do."""
    import torch
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    r = senmoe.Rows8(torch.zeros(4, 64, dtype=torch.uint8).view(torch.float8_e4m3fn),
                     torch.zeros(4, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    for call in (lambda: senmoe.quantize8(x), lambda: senmoe.quantize8(x.float()), lambda: senmoe.rms_norm(x, x[0]),
                 lambda: senmoe.rms_norm(x.float(), x[0]), lambda: senmoe.rms_norm_backward(x, x, x[0]),
                 lambda: senmoe.linear8(r, r), lambda: senmoe.linear8(x, r), lambda: senmoe.linear8(r, r, dtype=torch.float32),
                 lambda: senmoe.linear8((r.codes, r.scales), r), lambda: senmoe.linear8_input_grad(x, r),
                 lambda: senmoe.linear8_input_grad(x.float(), r)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: senmoe.linear8(r, r, activation="tanh"), lambda: senmoe.linear8_input_grad(x, r, activation="tanh"),
                 lambda: senmoe.grouped_linear8(r, r, None), lambda: senmoe.grouped_linear8_input_grad(x, r, None)):
        with pytest.raises(senmoe.SenMoeError) as e:
            call()
        assert e.value.status == BAD
    assert r.dequantize().shape == (4, 64) and r.take(torch.tensor([3, 0])).scales.shape == (2, 2)
