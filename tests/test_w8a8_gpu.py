"""The 8-bit quantiser (with and without residual + RMSNorm) and the int8 GEMM against fp64 on the CPU.

Codes: with u = 2^-24 (half a step of fp32) the kernel's z * (127 / max|z|) carries at most 5 roundings with a norm (h, z, the
maximum's two, the quotient, the product: 6 u) and 2 without, relative, so a code of at most 127 can only differ from the
exact one where the exact quotient lies within 127 * 6 u (127 * 2 u) of a half.  Scales: the sum of squares of at most 32
terms per thread plus ten tree steps is off by at most 43 u, its root by half of that, and the few products behind it by 6 u.
GEMM: the integer sum is exact; its conversion, the two products and the addition are off by at most 4 u of
|product| + |bias|, and the output by half a step of its type."""
import ctypes

import pytest
import torch

from nunchaku_b200 import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16]


def _rand(*shape, seed, dtype, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _exact(x, weight=None, residual=None, eps=1e-6):
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    y = h if weight is None else h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double()
    top = y.abs().amax(-1, keepdim=True)
    return y, top.squeeze(-1) / 127, torch.where(top > 0, y * 127 / top, torch.zeros_like(y))


def _check(got, x, weight=None, residual=None, eps=1e-6):
    codes, scales = got[0].cpu(), got[1].cpu()
    torch.cuda.synchronize()
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32 and codes.shape == x.shape and scales.shape == x.shape[:-1]
    _, scale, q = _exact(x, weight, residual, eps)
    near = 127 * (2 if weight is None else 6) * U
    assert ((codes.double() - q).abs() <= 0.5 + near).all()
    rel = (2 if weight is None else 28) * U
    assert ((scales.double() - scale).abs() <= rel * scale + 2.0 ** -149).all()
    if residual is not None:
        assert torch.equal(got[2].cpu(), (x.float() + residual.float()).to(x.dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 2240), (3, 128), (149, 256), (300, 272), (777, 1152), (1200, 2304), (150, 4112), (5, 12304), (200, 16384)])
def test_quantize(rows, cols, dtype):
    from nunchaku_b200.ops import quantize_w8a8

    x = _rand(rows, cols, seed=rows + cols, dtype=dtype, std=3.0)
    _check(quantize_w8a8(x.cuda()), x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 2240), (148, 64), (151, 768), (640, 2240), (160, 5600), (3, 16384), (150, 16384)])
def test_norm_and_quantize(rows, cols, residual, dtype):
    from nunchaku_b200.ops import rms_norm_quantize_w8a8

    x, w = _rand(rows, cols, seed=rows, dtype=dtype), _rand(cols, seed=cols, dtype=dtype, std=0.3) + 1
    r = _rand(rows, cols, seed=7, dtype=dtype, std=2.0) if residual else None
    got = rms_norm_quantize_w8a8(x.cuda(), w.cuda(), residual=None if r is None else r.cuda())
    assert (got[2] is None) == (r is None)
    _check(got, x, w, r)


def test_leading_dimensions_and_strided_rows():
    from nunchaku_b200.ops import quantize_w8a8, rms_norm_quantize_w8a8

    wide = _rand(4, 37, 3 * 256, seed=1, dtype=torch.bfloat16).cuda()
    part, res = wide[..., 256:512], wide[..., 512:]
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    before = wide.clone()
    _check(quantize_w8a8(part), part.cpu())
    _check(rms_norm_quantize_w8a8(part, w, residual=res), part.cpu(), w.cpu(), res.cpu())
    assert torch.equal(wide, before)


def test_rows_of_zeros_and_of_values_that_are_not_finite():
    from nunchaku_b200.ops import quantize_w8a8, rms_norm_quantize_w8a8

    for dtype in DTYPES:
        x = _rand(400, 512, seed=3, dtype=dtype)
        x[5] = 0
        x[17, 100], x[18, 511], x[19, 0] = float("nan"), float("inf"), float("-inf")
        w = torch.ones(512, dtype=dtype)
        bad = torch.zeros(400, dtype=torch.bool)
        bad[17:20] = True
        for got in (quantize_w8a8(x.cuda())[:2], rms_norm_quantize_w8a8(x.cuda(), w.cuda())[:2]):
            codes, scales = got[0].cpu(), got[1].cpu()
            assert torch.equal(scales.isnan(), bad) and (codes[bad] == 0).all()
            assert scales[5] == 0 and (codes[5] == 0).all()
            assert (codes[~bad].abs().amax(-1)[torch.arange(397) != 5] == 127).all()
    # squares beyond fp32: reported, not quietly zero
    x = torch.full((2, 64), 1e30, dtype=torch.bfloat16)
    x[1] = 1.0
    codes, scales, _ = rms_norm_quantize_w8a8(x.cuda(), torch.ones(64, dtype=torch.bfloat16, device="cuda"))
    assert scales[0].isnan().item() and (codes[0] == 0).all() and (codes[1] == 127).all()


def test_smallest_and_largest_magnitudes():
    from nunchaku_b200.ops import quantize_w8a8

    x = _rand(6, 256, seed=9, dtype=torch.float32)
    for k, s in enumerate([1e-38, 3e-39, 1e-36, 1e37, 1e-20, 1.0]):
        x[k] *= s
    x = x.to(torch.bfloat16)
    _check(quantize_w8a8(x.cuda()), x)
    y = torch.zeros(1, 64, dtype=torch.bfloat16)
    y[0, 3] = 2.0 ** -133   # the smallest bf16 number: the scale itself is below fp32's normal numbers
    codes, scales = quantize_w8a8(y.cuda())
    assert codes[0, 3] == 127 and codes.abs().sum() == 127


def test_ties_of_rows_up_to_the_largest_numbers():
    """values of half the row's largest stand on the tie 63.5 exactly: 64 (to even), whatever the row's magnitude"""
    from nunchaku_b200.ops import quantize_w8a8

    x = torch.zeros(254, 32, dtype=torch.bfloat16)
    x[:, 5] = torch.tensor([1.0 + k / 128 for k in range(127)] * 2).bfloat16() * torch.tensor([2.0 ** 126] * 127 + [2.0 ** -100] * 127).bfloat16()
    x[:, 6], x[:, 7] = x[:, 5] / 2, -x[:, 5] / 2
    codes, scales = quantize_w8a8(x.cuda())
    assert (codes[:, 5] == 127).all() and (codes[:, 6] == 64).all() and (codes[:, 7] == -64).all() and codes.float().abs().sum() == 254 * 255
    _check((codes, scales), x)


@pytest.mark.parametrize("onto", ["x", "residual"])
def test_residual_stream_in_place(onto):
    """through the C interface, hidden may be x or the residual"""
    x, r, w = (_rand(*s, seed=40 + i, dtype=torch.bfloat16).cuda() for i, s in enumerate([(3000, 2240), (3000, 2240), (2240,)]))
    from nunchaku_b200.ops import rms_norm_quantize_w8a8

    ref = rms_norm_quantize_w8a8(x, w, residual=r)
    codes, scales, hidden = torch.empty_like(ref[0]), torch.empty_like(ref[1]), x if onto == "x" else r
    args = _lib.QuantizeW8A8Args(x.data_ptr(), r.data_ptr(), w.data_ptr(), codes.data_ptr(), scales.data_ptr(), hidden.data_ptr(), 3000, 2240, 2240,
                                 2240, 1e-6, 0)
    _lib.check(_lib.load().svdq_quantize_w8a8(ctypes.byref(args), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(codes, ref[0]) and torch.equal(scales, ref[1]) and torch.equal(hidden, ref[2])


def test_two_calls_at_once():
    """on two streams, each call's result as when alone"""
    from nunchaku_b200.ops import gemm_w8a8, quantize_w8a8

    x = [_rand(M, 512, seed=30 + M, dtype=torch.bfloat16).cuda() for M in (3, 700)]
    w, sw = quantize_w8a8(_rand(264, 512, seed=33, dtype=torch.bfloat16).cuda())
    step = lambda t: gemm_w8a8(*(lambda c, s: (c, w, s))(*quantize_w8a8(t)), sw)
    ref = [step(t).clone() for t in x]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(x[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, r) for i, r in enumerate(ref) for g in got[i])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(16,), (1, 48), (3, 5, 272), (4000, 2240)])
def test_dequantize(shape, dtype):
    from nunchaku_b200.ops import dequantize_w8a8

    g = torch.Generator().manual_seed(len(shape))
    c = torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)
    s = torch.rand(shape[:-1], generator=g) * 0.1
    got = dequantize_w8a8(c.cuda(), s.cuda(), out_dtype=dtype).cpu()
    assert torch.equal(got, (c.float() * s[..., None]).to(dtype))
    for bad in ((c.cuda().half(), s.cuda()), (c.cuda(), s.cuda().double()), (c.cuda(), torch.zeros(*shape[:-1], 1, device="cuda"))):
        with pytest.raises(ValueError):
            dequantize_w8a8(*bad)


# ------------------------------------------------------------------------------------------------------------------ GEMM
def _gemm_case(M, N, K, seed, dtype, bias):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    sa, sw = torch.rand(M, generator=g) * 0.02 + 1e-3, torch.rand(N, generator=g) * 0.01 + 1e-4
    return a, w, sa, sw, (torch.randn(N, generator=g) * 3).to(dtype) if bias else None


def _gemm_check(got, a, w, sa, sw, b, dtype):
    torch.cuda.synchronize()
    assert _lib.device_status() == (0, 0)
    prod = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    exact = prod if b is None else prod + b.double()
    slack = 4 * U * (prod.abs() + (0 if b is None else b.double().abs()))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134      # half a step of the smallest numbers
    tol = slack + (exact.abs() + slack) * torch.finfo(dtype).eps / 2 + tiny
    got = got.cpu()
    assert got.dtype == dtype and got.shape == exact.shape
    assert ((got.double() - exact).abs() <= tol).all()


SHAPES = [(1, 8, 16), (1, 2240, 2240), (2, 128, 128), (16, 136, 400), (17, 264, 144), (33, 1000, 272), (64, 128, 1152), (65, 392, 2240),
          (128, 2304, 512), (129, 8, 16), (129, 200, 48), (256, 256, 128), (257, 264, 2240), (300, 4480, 656), (1000, 72, 1280), (2147, 640, 2240)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(M, N, K, dtype):
    from nunchaku_b200.ops import gemm_w8a8

    bias = (M + N) % 3 != 0
    case = _gemm_case(M, N, K, M + N + K, dtype, bias)
    a, w, sa, sw, b = [None if t is None else t.cuda() for t in case]
    _gemm_check(gemm_w8a8(a, w, sa, sw, bias=b, out_dtype=dtype), *case, dtype)


def test_gemm_many_tiles_per_pair():
    """more tiles than CTA pairs: accumulators and ring wrap around"""
    from nunchaku_b200.ops import gemm_w8a8

    case = _gemm_case(5000, 1864, 1040, 5, torch.bfloat16, True)
    got = gemm_w8a8(*[t.cuda() for t in case])
    _gemm_check(got, *case, torch.bfloat16)


def test_gemm_largest_sums():
    """the deepest K with every product 2^14: the sum reaches 2^31 - 2^18 and does not wrap"""
    from nunchaku_b200.ops import gemm_w8a8

    K = 131056
    for M in (3, 140):
        a = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
        w = torch.full((16, K), -128, dtype=torch.int8, device="cuda")
        w[1::2] = 127
        out = gemm_w8a8(a, w, torch.full((M,), 2.0 ** -20, device="cuda"), torch.full((16,), 2.0 ** -4, device="cuda"))
        exp = torch.tensor([2.0 ** 14 * K, -128.0 * 127 * K]).mul(2.0 ** -24).to(torch.bfloat16)
        assert torch.equal(out.cpu(), exp.repeat(M, 8))


@pytest.mark.parametrize("M", [5, 200])
def test_gemm_into_a_wider_buffer_leaves_the_rest(M):
    from nunchaku_b200.ops import gemm_w8a8

    case = _gemm_case(M, 200, 320, 9, torch.bfloat16, True)
    buf = torch.full((M + 3, 328), 7.0, dtype=torch.bfloat16, device="cuda")
    out = gemm_w8a8(*[t.cuda() for t in case], out=buf[:M, 64:264])
    _gemm_check(out, *case, torch.bfloat16)
    assert (buf[M:] == 7).all() and (buf[:, :64] == 7).all() and (buf[:, 264:] == 7).all()


def test_gemm_passes_a_bad_row_on_as_nan():
    from nunchaku_b200.ops import gemm_w8a8, quantize_w8a8

    x = _rand(40, 64, seed=2, dtype=torch.bfloat16)
    x[7, 3] = float("nan")
    w = _rand(24, 64, seed=3, dtype=torch.bfloat16)
    qa, sa = quantize_w8a8(x.cuda())
    qw, sw = quantize_w8a8(w.cuda())
    y = gemm_w8a8(qa, qw, sa, sw).cpu()
    assert y[7].isnan().all() and torch.isfinite(y[torch.arange(40) != 7].float()).all()


@pytest.mark.parametrize("M", [4, 300])
def test_on_another_stream_and_in_a_graph(M):
    from nunchaku_b200.ops import gemm_w8a8, rms_norm_quantize_w8a8

    x, w = _rand(M, 256, seed=4, dtype=torch.float16).cuda(), torch.ones(256, dtype=torch.float16, device="cuda")
    _, wgt, _, sw, b = [t.cuda() for t in _gemm_case(1, 264, 256, 6, torch.float16, True)]

    def step():
        c, s, h = rms_norm_quantize_w8a8(x, w, residual=x)
        return gemm_w8a8(c, wgt, s, sw, bias=b), h

    ref = [t.clone() for t in step()]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = step()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x.copy_(_rand(M, 256, seed=5, dtype=torch.float16))
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_python_layer_refuses():
    from nunchaku_b200.ops import gemm_w8a8, quantize_w8a8, rms_norm_quantize_w8a8

    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for bad in (x.float(), x[:, :24], x[:0], x.t(), x[:, :63]):
        with pytest.raises(ValueError):
            quantize_w8a8(bad)
    for kw in (dict(weight=w[:32]), dict(weight=w.half()), dict(weight=None), dict(weight=w, residual=x[:2]), dict(weight=w, residual=x.half()),
               dict(weight=w, eps=-1e-6), dict(weight=w, eps=float("nan"))):
        with pytest.raises(ValueError):
            rms_norm_quantize_w8a8(x, **kw)
    with pytest.raises(NotImplementedError):
        quantize_w8a8(torch.zeros(1, 16400, dtype=torch.bfloat16, device="cuda"))
    q, s = quantize_w8a8(x)
    ok = dict(act=q, wgt=q, ascales=s, wscales=s)
    wq, ws = torch.zeros(8, 64, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    ok.update(wgt=wq, wscales=ws)
    for kw in (dict(act=x), dict(act=q[:, :32]), dict(wgt=q[:3], wscales=s[:3]), dict(ascales=s[:3]), dict(wscales=s), dict(ascales=s.double()),
               dict(bias=w[:8].half(), out_dtype=torch.bfloat16), dict(bias=w[:7]), dict(out_dtype=torch.float32), dict(act=q[:0], ascales=s[:0]),
               dict(out=torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")), dict(out=torch.zeros(8, 4, dtype=torch.bfloat16, device="cuda").t()),
               dict(wgt=wq.cpu())):
        with pytest.raises(ValueError):
            gemm_w8a8(**{**ok, **kw})
    assert (gemm_w8a8(**ok) == 0).all()
