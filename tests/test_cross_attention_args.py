"""Argument checks of svdq_cross_attention (no GPU: they run before any CUDA call) and the C layout of its struct."""
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
    cname, cls = "svdq_cross_attention_args", lib.CrossAttentionArgs
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){", f'printf("size %zu\\n", sizeof({cname}));']
    member = lambda f: f"{f[:-1]}[{f[-1]}]" if "_stride" in f and f[-1].isdigit() else f   # q_stride0 stands for q_stride[0]
    lines += [f'printf("{f} %zu\\n", offsetof({cname}, {member(f)}));' for f, _ in cls._fields_]
    c = tmp_path / "layout.c"
    c.write_text("\n".join([*lines, "return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(c)], check=True)
    got = dict(l.split() for l in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.strip().splitlines())
    assert int(got["size"]) == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert int(got[f]) == getattr(cls, f).offset, f


GOOD = dict(q=64, k=64, v=64, out=64, q_stride=(4096, 64, 256), k_stride=(4096, 64, 256), v_stride=(4096, 64, 256), o_stride=(4096, 64, 256),
            batch=2, heads=4, kv_heads=4, q_len=16, kv_len=16, head_dim=64, scale=0.125)


def _call(lib, **kw):
    d = {**GOOD, **kw}
    for s in ("q_stride", "k_stride", "v_stride", "o_stride"):
        d.update({f"{s}{i}": x for i, x in enumerate(d.pop(s))})
    return lib.load().svdq_cross_attention(ctypes.byref(lib.CrossAttentionArgs(**d)), None)


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=8), dict(k=8), dict(v=8), dict(out=8), dict(batch=0),
                                 dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(q_len=0), dict(kv_len=0), dict(head_dim=0), dict(head_dim=12),
                                 dict(head_dim=136), dict(batch=65536), dict(heads=65536, kv_heads=65536), dict(scale=0.0), dict(scale=-1.0),
                                 dict(scale=float("inf")), dict(scale=float("nan")), dict(dtype=2), dict(kv_lens=64, mask=64), dict(kv_lens=64, kv_offsets=64),
                                 dict(kv_offsets=64, mask=64), dict(mask=64, mask_stride=-1), dict(kv_lens=2), dict(q_stride=(4096, 64, 252)),
                                 dict(k_stride=(4096, 68, 256)), dict(v_stride=(4100, 64, 256)), dict(q_stride=(4096, 64, 0)), dict(k_stride=(4096, 64, 56)),
                                 dict(o_stride=(0, 64, 256)), dict(o_stride=(4096, 0, 256)), dict(k_stride=(4096, -64, 256))])
def test_refuses(lib, bad):
    assert _call(lib, **bad) == lib.SVDQ_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("big", [dict(q_len=2 ** 30 + 1), dict(kv_len=2 ** 30 + 1), dict(kv_len=2 ** 31 - 1)])
def test_refuses_more_tokens_than_its_indices_count(lib, big):
    assert _call(lib, **big) == lib.SVDQ_ERR_INVALID_ARGUMENT


def test_refuses_null_and_a_mask_that_is_too_long(lib):
    assert lib.load().svdq_cross_attention(None, None) == lib.SVDQ_ERR_INVALID_ARGUMENT
    assert _call(lib, mask=64, mask_stride=70000, kv_len=32769) == lib.SVDQ_ERR_UNSUPPORTED


def test_python_layer_refuses_cpu_tensors():
    from nunchaku_b200.ops import cross_attention

    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        cross_attention(q, q, q)
