"""Cross attention against fp64 softmax attention on the CPU.

Tolerance, per output element o = sum_i p_i v_i / sum_i p_i with A = sum_i p_i |v_i| / sum_i p_i: the probabilities are rounded to the
16-bit type (half a step: eps / 2 relative), a quarter of the exponentials is a cubic good to 7.6e-5 (it acts on p and on the sum),
a score is off by at most d = (D + 3) 2^-24 scale max_i sum_c |q_c k_c| (fp32 accumulation over D channels, scale, exponent), which moves
p and the sum; the fp32 sums over blocks, warps and CTAs add less than 2^-16.  fp16 probabilities below 2^-14 lose at most 2^-25
each, against a sum of at least 1 (the maximum in use is one of the row's own scores and never above the largest).  The output itself: half a step of o."""
import pytest
import torch

from nunchaku_b200 import _lib

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _keep(B, T, kv_lens=None, mask=None):
    if mask is not None:
        return mask.cpu()
    if kv_lens is not None:
        return torch.arange(T) < kv_lens.cpu().clamp(0, T)[:, None]
    return torch.ones(B, T, dtype=torch.bool)


def _exact(q, k, v, keep, scale):
    """q [B, H, Tq, D], k, v [B, Hk, T, D], keep [B, T]; returns the output and its tolerance, both [B, Tq, H*D] in fp64."""
    B, H, Tq, D = q.shape
    eps = torch.finfo(q.dtype).eps
    out, tol = torch.zeros(B, Tq, H, D, dtype=torch.float64), torch.zeros(B, Tq, H, D, dtype=torch.float64)
    group = H // k.shape[1]
    for b in range(B):
        idx = keep[b].nonzero().squeeze(1)
        if len(idx) == 0:
            continue
        kb, vb = k[b][:, idx].double().repeat_interleave(group, 0), v[b][:, idx].double().repeat_interleave(group, 0)
        qb = q[b].double()
        w = torch.softmax(scale * (qb @ kb.transpose(1, 2)), dim=-1)
        d = (D + 3) * 2.0 ** -24 * scale * (qb.abs() @ kb.abs().transpose(1, 2)).amax(-1, keepdim=True)
        o, a = w @ vb, w @ vb.abs()
        t = a * (eps / 2 + 2 * 7.6e-5 + 2.0 ** -16 + 2 * d) + o.abs() * eps / 2
        if q.dtype == torch.float16:
            t += 2.0 ** -25 * vb.abs().sum(1, keepdim=True) + 2.0 ** -25
        out[b], tol[b] = o.transpose(0, 1), t.transpose(0, 1) + 1e-30
    return out.reshape(B, Tq, H * D), tol.reshape(B, Tq, H * D)


def _check(got, q, k, v, keep, scale):
    torch.cuda.synchronize()
    assert _lib.device_status() == (0, 0)
    exp, tol = _exact(q.cpu(), k.cpu(), v.cpu(), keep, scale)
    got = got.cpu()
    assert got.shape == exp.shape and got.dtype == q.dtype
    err = (got.double() - exp).abs()
    assert (err <= tol).all(), f"largest error over tolerance {(err / tol).max().item()}"
    assert (got[~keep.any(1)] == 0).all()


def _inputs(B, H, Hk, Tq, T, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Tq, H, D, generator=g).to(dtype).cuda().transpose(1, 2)
    kv = torch.randn(B, T, 2, Hk, D, generator=g).to(dtype).cuda()
    return q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)


# few query rows, one tile, ragged tiles; one state, ragged blocks, exact blocks, many blocks; head widths of every step count
SIZES = [(1, 1, 1, 1, 1, 8), (1, 20, 20, 1, 300, 112), (3, 4, 2, 1, 65, 128), (2, 6, 2, 5, 129, 40), (2, 2, 2, 16, 64, 64), (1, 3, 1, 2, 1000, 72),
         (1, 2, 2, 17, 1, 16), (2, 3, 3, 128, 128, 64), (1, 4, 2, 129, 300, 112), (2, 2, 1, 33, 77, 8), (1, 2, 2, 300, 16, 128), (2, 2, 2, 200, 257, 96),
         (1, 2, 1, 64, 190, 24), (1, 1, 1, 100, 1153, 80), (3, 1, 1, 40, 64, 48), (1, 2, 2, 70, 192, 104),
         # row tiles of 16 over long lists, split; many heads: 128-row tiles over several blocks (which of the two runs goes by their times)
         (1, 4, 2, 40, 1000, 72), (2, 6, 2, 30, 700, 128), (1, 1, 1, 500, 900, 32), (1, 16, 16, 140, 300, 112), (1, 16, 4, 150, 257, 128),
         (2, 32, 32, 150, 300, 64), (2, 32, 8, 129, 520, 40), (4, 40, 40, 20, 200, 96),
         # more 128-row tiles than there are places: two at a time over the same states, of one head or of two that share a stored one
         (2, 80, 80, 150, 300, 112), (1, 160, 80, 129, 130, 72), (3, 60, 60, 256, 64, 128), (1, 310, 155, 100, 200, 24), (5, 20, 20, 500, 65, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hk,Tq,T,D", SIZES)
def test_all_states(B, H, Hk, Tq, T, D, dtype):
    from nunchaku_b200.ops import cross_attention

    q, k, v = _inputs(B, H, Hk, Tq, T, D, dtype, seed=Tq + T + D)
    _check(cross_attention(q, k, v), q, k, v, _keep(B, T), D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq", [1, 5, 150])
@pytest.mark.parametrize("H,Hk,T,D", [(2, 2, 300, 112), (4, 2, 128, 64), (3, 3, 700, 128), (2, 1, 40, 32), (18, 18, 300, 112), (20, 10, 200, 24)])
def test_lengths_with_nan_behind_them(Tq, H, Hk, T, D, dtype):
    from nunchaku_b200.ops import cross_attention

    lens = torch.tensor([0, 1, T, T - 3, min(T, 64), min(T, 129), 17, T + 50, -4], dtype=torch.int32)   # the last two are clamped
    B = len(lens)
    q, k, v = _inputs(B, H, Hk, Tq, T, D, dtype, seed=T + Tq)
    keep = _keep(B, T, kv_lens=lens)
    ck, cv = k.clone(), v.clone()
    hidden = ~keep.cuda()[:, None, :, None]
    k.masked_fill_(hidden, float("nan"))
    v.masked_fill_(hidden, float("inf"))
    got = cross_attention(q, k, v, kv_lens=lens.cuda())
    _check(got, q, ck, cv, keep, D ** -0.5)
    v.masked_fill_(hidden, float("nan"))
    k.masked_fill_(hidden, torch.finfo(dtype).min)
    assert torch.equal(cross_attention(q, k, v, kv_lens=lens.cuda()), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq", [1, 3, 140, 300])
@pytest.mark.parametrize("H,Hk,T,D", [(2, 2, 77, 64), (2, 1, 520, 112), (1, 1, 1, 128), (4, 4, 300, 32), (22, 22, 200, 64), (24, 12, 450, 96)])
def test_masks(Tq, H, Hk, T, D, dtype):
    from nunchaku_b200.ops import cross_attention

    g = torch.Generator().manual_seed(T)
    mask = torch.rand(7, T, generator=g) < 0.6
    mask[0] = True
    mask[1] = False                                  # no states
    mask[2] = False
    mask[2, T - 1] = True                            # only the last: the blocks before it are skipped
    mask[3] = False
    mask[3, 0] = True
    mask[4, 64 if T > 64 else 0:] = False            # leading states only
    if T > 400:
        mask[5, 100:400] = False                     # empty blocks between others
    B = len(mask)
    q, k, v = _inputs(B, H, Hk, Tq, T, D, dtype, seed=T + Tq)
    ck, cv = k.clone(), v.clone()
    hidden = ~mask.cuda()[:, None, :, None]
    k.masked_fill_(hidden, float("inf"))
    v.masked_fill_(hidden, float("nan"))
    wide = torch.ones(B, T + 5, dtype=torch.bool, device="cuda")
    wide[:, :T] = mask.cuda()
    _check(cross_attention(q, k, v, mask=wide[:, :T]), q, ck, cv, mask, D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq", [1, 6, 200])
@pytest.mark.parametrize("H,Hk,D", [(2, 2, 112), (4, 2, 64), (3, 1, 128), (20, 20, 112), (20, 10, 40)])
def test_packed(Tq, H, Hk, D, dtype):
    from nunchaku_b200.ops import cross_attention

    lens = [300, 0, 5, 128, 1, 64, 0, 213]
    B, T = len(lens), max(lens)
    off = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    q, kp, vp = _inputs(B, H, Hk, Tq, T, D, dtype, seed=Tq + D)
    keep = _keep(B, T, kv_lens=torch.tensor(lens))
    total = sum(lens)
    packed = torch.full((total + 9, 2, Hk, D), float("nan"), dtype=dtype, device="cuda")   # rows behind the last sample: NaN
    for b, n in enumerate(lens):
        packed[off[b]:off[b] + n, 0] = kp[b, :, :n].transpose(0, 1)
        packed[off[b]:off[b] + n, 1] = vp[b, :, :n].transpose(0, 1)
    got = cross_attention(q, packed[:, 0], packed[:, 1], kv_offsets=off.cuda())
    _check(got, q, kp, vp, keep, D ** -0.5)
    packed[off[3]:off[4]] = float("nan")             # one sample's states: nobody else's business
    again = cross_attention(q, packed[:, 0], packed[:, 1], kv_offsets=off.cuda())
    others = [b for b in range(B) if b != 3]
    assert torch.equal(again[others], got[others]) and again[3].isnan().all()
    # offsets that point outside are clamped to the rows there are
    bad = off.clone()
    bad[-1] = total + 1000
    full = cross_attention(q, packed[:total, 0], packed[:total, 1], kv_offsets=bad.cuda())
    assert torch.equal(full[others], got[others])
    bad = torch.tensor([-5, -1, 4, 2, 10 ** 9, 2 ** 31 - 1, -2 ** 31, 0, 3], dtype=torch.int32)
    assert torch.isfinite(cross_attention(q, packed[:total, 0], packed[:total, 1], kv_offsets=bad.cuda())[[0, 2]]).all()
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("Tq,H", [(2, 4), (130, 4), (130, 32), (130, 100)])
def test_layouts(Tq, H):
    """head-major, token-major, broadcast over batch or heads, an output inside a wider buffer"""
    from nunchaku_b200.ops import cross_attention

    B, T, D = 2, 150, 64
    g = torch.Generator().manual_seed(3)
    q = torch.randn(B, H, Tq, D, generator=g).bfloat16().cuda()
    k1, v1 = (torch.randn(1, H, T, D, generator=g).bfloat16().cuda() for _ in range(2))
    keep, s = _keep(B, T), D ** -0.5
    k, v = k1.expand(B, H, T, D), v1.expand(B, H, T, D)
    _check(cross_attention(q, k, v), q, k, v, keep, s)
    k, v = k1[:, :1].expand(B, H, T, D), v1[:, :1].expand(B, H, T, D)
    ref = cross_attention(q, k, v)
    _check(ref, q, k, v, keep, s)
    assert torch.equal(cross_attention(q, k[:, :1], v[:, :1]), ref)          # one stored head for all
    buf = torch.full((B, Tq + 7, H * D + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, 3:3 + Tq, 32:32 + H * D]
    assert cross_attention(q, k, v, out=out) is out
    assert torch.equal(out, ref) and (buf[:, :3] == 7).all() and (buf[:, 3 + Tq:] == 7).all() and (buf[:, :, :32] == 7).all() and (buf[:, :, 32 + H * D:] == 7).all()
    hm = torch.empty(B, H, Tq, D, dtype=torch.bfloat16, device="cuda")
    cross_attention(q, k, v, out=hm)
    assert torch.equal(hm.transpose(1, 2).reshape(B, Tq, H * D), ref)


@pytest.mark.parametrize("Tq,H", [(1, 2), (150, 2), (150, 16), (150, 80)])
def test_growing_scores_and_large_scale(Tq, H):
    """the maximum rises from block to block by far more than the rescaling step; nearly one-hot weights"""
    from nunchaku_b200.ops import cross_attention

    B, T, D = 2, 900, 128
    g = torch.Generator().manual_seed(8)
    q = torch.randn(B, H, Tq, D, generator=g).abs().bfloat16().cuda()
    k = (torch.randn(B, H, T, D, generator=g).abs() * torch.linspace(0.05, 3, T)[:, None]).bfloat16().cuda()
    v = torch.randn(B, H, T, D, generator=g).bfloat16().cuda()
    for s in (D ** -0.5, 0.5):
        _check(cross_attention(q, k, v, scale=s), q, k, v, _keep(B, T), s)
    k = k.flip(2)                                    # and falls
    _check(cross_attention(q, k, v, scale=0.5), q, k, v, _keep(B, T), 0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq,H", [(3, 2), (140, 32), (140, 80)])
def test_a_bad_state_that_is_to_be_seen_is_not_hidden(Tq, H, dtype):
    """a NaN in one state of K (at every place of a block in turn) or V shows in every row that sees it, and nowhere else"""
    from nunchaku_b200.ops import cross_attention

    B, T, D = 2, 100, 64
    for part in (1, 2):
        for at in range(0, T, 1 if Tq == 3 else 5):
            qkv = _inputs(B, H, H, Tq, T, D, dtype, seed=at)
            if at == 0:
                clean = [cross_attention(*_inputs(B, H, H, Tq, T, D, dtype, seed=s)) for s in range(T)]
            qkv[part][1, H - 1, at, 7] = float("nan")
            got = cross_attention(*qkv)
            bad = got.isnan()
            assert bad[1, :, (H - 1) * D + 7].all() and (part == 2 or bad[1, :, (H - 1) * D:].all())
            bad[1, :, (H - 1) * D + 7] = False
            if part == 1:
                bad[1, :, (H - 1) * D:] = False
            assert not bad.any()
            assert torch.equal(got[0], clean[at][0]) and torch.equal(got[1, :, :(H - 1) * D], clean[at][1, :, :(H - 1) * D])


@pytest.mark.parametrize("Tq,H", [(3, 2), (140, 32), (140, 160)])
def test_states_of_minus_infinity(Tq, H):
    """scores of -inf (whole blocks of them, ahead of others and behind) weigh nothing"""
    from nunchaku_b200.ops import cross_attention

    B, T, D = 1, 300, 64
    q, k, v = _inputs(B, H, H, Tq, T, D, torch.bfloat16, seed=3)
    q = q.abs() + 0.25
    keep = torch.ones(B, T, dtype=torch.bool)
    for lo, hi in ((0, 70), (0, 1), (100, 260), (299, 300)):
        k2 = k.clone()
        k2[:, :, lo:hi] = -float("inf")
        keep2 = keep.clone()
        keep2[:, lo:hi] = False
        k3 = k.clone()
        _check(cross_attention(q, k2, v), q, k3, v, keep2, D ** -0.5)


@pytest.mark.parametrize("Tq,H", [(3, 2), (140, 32), (140, 160)])
@pytest.mark.parametrize("masked", [False, True])
def test_scores_of_the_largest_magnitudes(Tq, H, masked):
    """scores down to -1e37: the state of the largest alone is seen, wherever it stands"""
    from nunchaku_b200.ops import cross_attention

    T, D = 200, 64
    q = torch.full((1, H, Tq, D), 2.0 ** 61, dtype=torch.bfloat16, device="cuda")
    v = torch.randn(1, H, T, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    mask = torch.ones(1, T, dtype=torch.bool, device="cuda")
    for at in (0, 63, 64, 130, 199):
        k = torch.full((1, H, T, D), -2.0 ** 60, dtype=torch.bfloat16, device="cuda")
        k[:, :, at] = -2.0 ** 59
        if masked:
            mask[:] = True
            mask[0, :64] = at < 64          # a first block of which nothing is to be seen
        got = cross_attention(q, k, v, mask=mask if masked else None)
        assert torch.equal(got.view(1, Tq, H, D), v[:, :, at][:, None].expand(1, Tq, H, D))


def test_two_calls_at_once():
    """on two streams, each call's result as when alone"""
    from nunchaku_b200.ops import cross_attention

    cases = [_inputs(2, 4, 4, 1, 900, 112, torch.bfloat16, seed=1), _inputs(2, 20, 20, 300, 300, 112, torch.bfloat16, seed=2),
             _inputs(2, 20, 20, 300, 300, 112, torch.bfloat16, seed=3), _inputs(2, 80, 80, 256, 300, 112, torch.bfloat16, seed=4)]
    ref = [cross_attention(*c).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(cross_attention(*cases[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, r) for i, r in enumerate(ref) for g in got[i])


def test_heads_and_samples_of_one_buffer():
    """q, k, v expanded over samples and heads (stride 0)"""
    from nunchaku_b200.ops import cross_attention

    for Tq, H in ((2, 4), (140, 32), (140, 64)):
        q, k, v = _inputs(1, 1, 1, Tq, 130, 72, torch.bfloat16, seed=5)
        got = cross_attention(q.expand(3, H, -1, -1), k.expand(3, H, -1, -1), v.expand(3, H, -1, -1))
        one = cross_attention(q.expand(3, H, -1, -1).contiguous(), k.expand(3, H, -1, -1).contiguous(), v.expand(3, H, -1, -1).contiguous())
        assert torch.equal(got, one)
        _check(got[:, :, :72], q.expand(3, 1, -1, -1), k.expand(3, 1, -1, -1), v.expand(3, 1, -1, -1), _keep(3, 130), 72 ** -0.5)


def test_long_state_lists():
    from nunchaku_b200.ops import cross_attention

    for Tq, T, H in ((1, 40000, 2), (200, 5000, 2), (130, 3000, 64)):
        q, k, v = _inputs(1, H, H // 2, Tq, T, 64, torch.bfloat16, seed=T)
        _check(cross_attention(q, k, v), q, k, v, _keep(1, T), 0.125)


def test_many_queries_over_millions_of_states():
    """longer lists than the tile kernel takes.  Tolerance: every row's sums run through up to T / 32 additions in fp32 per lane and product,
    each off by at most 2^-23 (the tensor cores may truncate), on top of the output's half step and the probabilities' (values are positive)"""
    from nunchaku_b200.ops import cross_attention

    T, Tq, D = 2 ** 22 + 100, 20480, 8
    g = torch.Generator().manual_seed(3)
    q = torch.randn(1, 1, Tq, D, generator=g).half().cuda()
    k = torch.randn(1, 1, T, D, generator=g).half().cuda()
    v = (torch.linspace(0, 2, T)[:, None] * torch.linspace(0.5, 1, D)).half()[None, None].cuda()
    got = cross_attention(q, k, v)
    torch.cuda.synchronize()
    assert _lib.device_status() == (0, 0)
    rows = [0, 777, Tq - 1]
    w = torch.softmax(D ** -0.5 * (q[0, 0, rows].double() @ k[0, 0].double().T), dim=-1)
    exp = w @ v[0, 0].double()
    assert ((got[0, rows].double() - exp).abs() <= exp * (2 * (T / 32) * 2.0 ** -23 + 2.0 ** -10)).all()
    with pytest.raises(NotImplementedError):
        cross_attention(torch.empty(1, 1, 2 ** 20, 8, dtype=torch.float16, device="cuda"), k, v)


def test_states_beyond_32_bit_offsets():
    """a batch whose last sample starts more than 2^31 elements into the buffer"""
    from nunchaku_b200.ops import cross_attention

    T, Hk, D, B = 4096, 8, 128, 2
    stride = 2 ** 31 + 2 ** 20
    buf = torch.zeros(stride + T * Hk * D, dtype=torch.bfloat16, device="cuda")
    k = buf.as_strided((B, Hk, T, D), (stride, D, Hk * D, 1))
    g = torch.Generator(device="cuda").manual_seed(1)
    k.copy_(torch.randn(B, Hk, T, D, generator=g, device="cuda"))
    for Tq in (1, 20):
        q = torch.randn(B, Hk, Tq, D, generator=g, device="cuda").bfloat16()
        got = cross_attention(q[:, :2], k[:, :2], k[:, :2])
        _check(got, q[:, :2], k[:, :2].contiguous(), k[:, :2].contiguous(), _keep(B, T), D ** -0.5)


@pytest.mark.parametrize("Tq", [1, 200])
def test_stream_and_graph(Tq):
    from nunchaku_b200.ops import cross_attention

    q, k, v = _inputs(2, 4, 4, Tq, 300, 112, torch.float16, seed=2)
    lens = torch.tensor([300, 123], dtype=torch.int32, device="cuda")
    ref = cross_attention(q, k, v, kv_lens=lens).clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = cross_attention(q, k, v, kv_lens=lens)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = cross_attention(q, k, v, kv_lens=lens)
    lens.copy_(torch.tensor([7, 0], dtype=torch.int32))     # read on the device at replay
    g.replay()
    assert torch.equal(out, cross_attention(q, k, v, kv_lens=lens)) and (out[1] == 0).all() and not torch.equal(out, ref)


@pytest.mark.parametrize("form", ["lens", "mask", "packed"])
def test_more_samples_than_one_launch_holds(form):
    from nunchaku_b200.ops import cross_attention

    B, H, Tq, T, D = 1600, 1, 17, 70, 16
    q, k, v = _inputs(B, H, H, Tq, T, D, torch.bfloat16, seed=12)
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    keep = _keep(B, T, kv_lens=lens)
    if form == "lens":
        got = cross_attention(q, k, v, kv_lens=lens.cuda())
    elif form == "mask":
        keep = torch.rand(B, T, generator=g) < 0.3
        keep[7] = False
        got = cross_attention(q, k, v, mask=keep.cuda())
    else:
        rows = keep.flatten().nonzero().squeeze(1).cuda()
        off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32).cuda()
        flat = lambda t: t.transpose(1, 2).reshape(B * T, H, D)[rows].contiguous()
        got = cross_attention(q, flat(k), flat(v), kv_offsets=off)
    _check(got, q, k, v, keep, D ** -0.5)


def test_python_layer_refuses():
    from nunchaku_b200.ops import cross_attention

    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")
    q, k = z(2, 4, 8, 64), z(2, 2, 10, 64)
    lens, off, mask = z(2, dtype=torch.int32), z(3, dtype=torch.int32), z(2, 10, dtype=torch.bool)
    assert (cross_attention(q, k, k) == 0).all()
    for a, kw in [((q.float(), k, k), {}), ((q, k.half(), k), {}), ((q, k, k[:, :, :5]), {}), ((q, z(1, 2, 10, 64), z(1, 2, 10, 64)), {}),
                  ((q, z(2, 3, 10, 64), z(2, 3, 10, 64)), {}), ((q, z(2, 2, 10, 32), z(2, 2, 10, 32)), {}), ((z(2, 4, 8, 136), z(2, 2, 10, 136), z(2, 2, 10, 136)), {}),
                  ((z(2, 4, 8, 12), z(2, 2, 10, 12), z(2, 2, 10, 12)), {}), ((q[..., ::2], k[..., ::2], k[..., ::2]), {}), ((q, k[:, :, :0], k[:, :, :0]), {}),
                  ((q, k, k), dict(scale=0.0)), ((q, k, k), dict(scale=-1.0)), ((q, k, k), dict(kv_lens=lens.long())), ((q, k, k), dict(kv_lens=lens[:1])),
                  ((q, k, k), dict(kv_lens=lens.cpu())), ((q, k, k), dict(mask=mask[:, :9])), ((q, k, k), dict(mask=mask.int())),
                  ((q, k, k), dict(mask=mask, kv_lens=lens)), ((q, k, k), dict(kv_offsets=off)), ((q, k[0].transpose(0, 1), k[0].transpose(0, 1)), dict(kv_offsets=off[:2])),
                  ((q, k, k), dict(out=z(2, 8, 128))), ((q, k, k), dict(out=z(2, 8, 256, dtype=torch.float16))), ((q, k, k), dict(out=z(1, 8, 256).expand(2, 8, 256)))]:
        with pytest.raises(ValueError):
            cross_attention(*a, **kw)
    with pytest.raises(NotImplementedError):
        cross_attention(q, z(2, 2, 32769, 64), z(2, 2, 32769, 64), mask=z(2, 32769, dtype=torch.bool))
    assert _lib.device_status() == (0, 0)
