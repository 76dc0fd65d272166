"""Argument checks of the 8-bit entry points (no GPU: they run before any CUDA call) and the C layout of their structs."""
import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "svdq_b200.h")


@pytest.fixture(scope="module")
def lib():
    from nunchaku_b200.csrc.build import build

    build()
    from nunchaku_b200 import _lib

    return _lib


def test_struct_layout_matches_c(lib, tmp_path):
    structs = {"svdq_quantize_w8a8_args": lib.QuantizeW8A8Args, "svdq_gemm_w8a8_args": lib.GemmW8A8Args,
               "svdq_dequantize_w8a8_args": lib.DequantizeW8A8Args}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    c = tmp_path / "layout.c"
    c.write_text("\n".join([*lines, "return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(c)], check=True)
    got = dict(l.split() for l in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.strip().splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"


def _q(lib, **kw):
    d = dict(x=64, codes=64, scales=64, rows=3, x_stride=64, cols=64, eps=1e-6)
    return lib.QuantizeW8A8Args(**{**d, **kw})


@pytest.mark.parametrize("bad", [dict(x=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(cols=0), dict(cols=24), dict(cols=-16),
                                 dict(x_stride=56), dict(x_stride=65), dict(x=8), dict(codes=8), dict(scales=2), dict(residual=64, weight=64),
                                 dict(hidden=64), dict(residual=64, hidden=64), dict(dtype=2),
                                 dict(residual=64, hidden=64, weight=64, residual_stride=0),
                                 dict(residual=72, hidden=64, weight=64, residual_stride=64), dict(weight=64, eps=-1.0),
                                 dict(weight=64, eps=float("nan"))])
def test_quantiser_refuses(lib, bad):
    assert lib.load().svdq_quantize_w8a8(ctypes.byref(_q(lib, **bad)), None) == lib.SVDQ_ERR_INVALID_ARGUMENT


def test_more_rows_than_an_int_counts_and_an_eps_of_zero(lib):
    assert lib.load().svdq_quantize_w8a8(ctypes.byref(_q(lib, weight=64, eps=0.0)), None) == lib.SVDQ_ERR_INVALID_ARGUMENT
    for big in (dict(M=2 ** 30 + 1), dict(N=2 ** 30 + 8, out_stride=2 ** 31)):
        d = dict(act=64, wgt=64, ascales=64, wscales=64, out=64, out_stride=16, M=1, N=16, K=64)
        assert lib.load().svdq_gemm_w8a8(ctypes.byref(lib.GemmW8A8Args(**{**d, **big})), None) == lib.SVDQ_ERR_INVALID_ARGUMENT


def test_w8a8_linear_refuses_sizes_its_operators_do_not_take():
    from nunchaku_b200.models import W8A8Linear

    for k, n in ((24, 16), (16400, 16), (32, 12)):
        with pytest.raises(ValueError):
            W8A8Linear(k, n)


def test_quantiser_refuses_null_and_too_wide(lib):
    assert lib.load().svdq_quantize_w8a8(None, None) == lib.SVDQ_ERR_INVALID_ARGUMENT
    assert lib.load().svdq_quantize_w8a8(ctypes.byref(_q(lib, cols=16400, x_stride=16400)), None) == lib.SVDQ_ERR_UNSUPPORTED
    assert b"16384" in lib.load().svdq_last_error_string()


@pytest.mark.parametrize("bad", [dict(codes=None), dict(scales=None), dict(out=None), dict(rows=0), dict(cols=8), dict(out=8), dict(dtype=3)])
def test_dequantiser_refuses(lib, bad):
    d = dict(codes=64, scales=64, out=64, rows=2, cols=32)
    assert lib.load().svdq_dequantize_w8a8(ctypes.byref(lib.DequantizeW8A8Args(**{**d, **bad})), None) == lib.SVDQ_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("bad", [dict(act=None), dict(wgt=None), dict(ascales=None), dict(wscales=None), dict(out=None), dict(M=0), dict(N=0),
                                 dict(N=12), dict(K=0), dict(K=24), dict(K=131072), dict(out_stride=8), dict(out_stride=20), dict(act=8), dict(wgt=8),
                                 dict(out=8), dict(ascales=2), dict(wscales=2), dict(bias=1), dict(dtype=-1)])
def test_gemm_refuses(lib, bad):
    d = dict(act=64, wgt=64, ascales=64, wscales=64, out=64, out_stride=16, M=1, N=16, K=64)
    assert lib.load().svdq_gemm_w8a8(ctypes.byref(lib.GemmW8A8Args(**{**d, **bad})), None) == lib.SVDQ_ERR_INVALID_ARGUMENT


def test_python_layer_refuses_cpu_tensors():
    from nunchaku_b200.ops import gemm_w8a8, quantize_w8a8, rms_norm_quantize_w8a8

    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        quantize_w8a8(x)
    with pytest.raises(ValueError):
        rms_norm_quantize_w8a8(x, x[0])
    with pytest.raises(ValueError):
        gemm_w8a8(x.to(torch.int8), x.to(torch.int8), torch.zeros(2), torch.zeros(2))


def test_rows_of_strided_tensors():
    from nunchaku_b200.ops.w8a8 import _rows

    t = torch.zeros(4, 6, 64)
    assert _rows("t", t, 64) == (24, 64)
    assert _rows("t", t[:, :, :32], 32) == (24, 64)
    assert _rows("t", t[:, 2], 64) == (4, 384)
    assert _rows("t", t[1:2, 2:3, :48], 48) == (1, 48)
    for bad in (t.transpose(0, 1), t[:, :5, :32], t.transpose(1, 2), t[0, 0].expand(3, 64)):
        with pytest.raises(ValueError):
            _rows("t", bad, bad.shape[-1])
