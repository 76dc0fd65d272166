"""Timed cases of four operators of a transformer's serving path, with their plain forms.

    rms_norm_quantize_w8a8   (x [+ residual]) -> RMSNorm -> 8-bit codes with one scale per token
    quantize_w8a8            x -> 8-bit codes with one scale per token
    gemm_w8a8                8-bit codes x 8-bit weights -> 16-bit, scales per token and per output channel, bias
    cross_attention          softmax attention of queries over an encoder's states of another length

``run`` computes the plain form (elementary torch operations in fp32, one rounding at the end) unless ``own`` is set;
then it makes the calls a user of the library makes.  ``exact`` restates each definition in fp64.  Codes are returned as
the values they stand for (code x scale, in the input's 16-bit type).
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a 2240-wide transformer between two layers: the residual's addition, the norm and the codes; latency only
        dict(name="norm_token", op="norm", rows=1, cols=2240, dtype="bf16", residual=True),
        # the caption states of a ragged batch of eight, normalised and quantised once for every block's key / value projection
        dict(name="norm_caption", op="norm", rows=2147, cols=2304, dtype="fp16", residual=False),
        # 32 images of 1024 tokens in a 2240-wide model: the bandwidth end
        dict(name="norm_images", op="norm", rows=32768, cols=2240, dtype="bf16", residual=True),
        # the conditioning vectors of a small batch in front of a modulation projection
        dict(name="quant_vectors", op="quant", rows=7, cols=1152, dtype="fp16"),
        # the hidden activations of a 5600-wide feed-forward layer
        dict(name="quant_hidden", op="quant", rows=18433, cols=5600, dtype="bf16"),
        # the modulation projection of eight images: every weight is read for eight rows
        dict(name="gemm_vectors", op="gemm", rows=8, k=2240, n=13440, dtype="bf16", bias=True),
        # key / value projection of a ragged batch of captions
        dict(name="gemm_caption", op="gemm", rows=2147, k=2240, n=4480, dtype="fp16", bias=True),
        # the expanding projection of a feed-forward layer over fifteen images of 1024 tokens and one
        dict(name="gemm_hidden", op="gemm", rows=15361, k=2240, n=11200, dtype="bf16", bias=False),
        # one query over one caption of 300 states, 20 heads of 112: latency only
        dict(name="cross_token", op="cross", batch=1, q_len=1, kv_len=300, heads=20, kv_heads=20, dim=112, dtype="bf16", form="full"),
        # single queries of sixteen sequences over long encoder outputs of their own lengths, 24 heads over 8 stored ones
        dict(name="cross_step", op="cross", batch=16, q_len=1, kv_len=4096, heads=24, kv_heads=8, dim=128, dtype="fp16", form="lens"),
        # queries of a small model over text states with a padding mask (with holes)
        dict(name="cross_mask", op="cross", batch=6, q_len=1000, kv_len=77, heads=16, kv_heads=16, dim=64, dtype="fp16", form="mask"),
        # 32 images of 1024 tokens over packed captions of up to 300 states, 20 heads of 112
        dict(name="cross_images", op="cross", batch=32, q_len=1024, kv_len=300, heads=20, kv_heads=20, dim=112, dtype="bf16", form="packed"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "quant", "gemm", "gemm", "cross", "cross", "cross"])
    dtype = rng.choice(["bf16", "fp16"])
    if op in ("norm", "quant"):
        cols = 16 * rng.randint(8, 350)
        rows = _log_int(rng, 1, 32768 * 2240 // cols)
        case = dict(op=op, rows=rows, cols=cols, dtype=dtype)
        if op == "norm":
            case["residual"] = rng.random() < 0.5
        return case
    if op == "gemm":
        k = 16 * rng.randint(8, 350)
        n = 8 * _log_int(rng, 16, 1680)
        rows = _log_int(rng, 1, min(16384, 15361 * 2240 * 11200 // (k * n)))
        return dict(op="gemm", rows=rows, k=k, n=n, dtype=dtype, bias=rng.random() < 0.7)
    heads = rng.choice([4, 8, 12, 16, 20, 24])
    kv_heads = rng.choice([h for h in range(1, heads + 1) if heads % h == 0] + [heads, heads])
    dim = rng.choice([32, 40, 64, 72, 80, 96, 112, 128])
    kv_len = _log_int(rng, 1, 4096)
    most = 32 * 1024 * 300 * 20 * 112 // (kv_len * heads * dim)
    q_len = min(most, rng.choice([1, _log_int(rng, 1, 2048), _log_int(rng, 16, 4096)]))
    most //= q_len
    states = 16 * 4096 * 8 * 128 // (kv_len * kv_heads * dim)
    batch = _log_int(rng, 1, max(1, min(32, most, states)))
    return dict(op="cross", batch=batch, q_len=q_len, kv_len=kv_len, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                form=rng.choice(["full", "lens", "mask", "packed"]))


def _lengths(case):
    """Valid encoder states per sample: one sample has all of them, the others between a tenth and all, now and then none."""
    B, T = case["batch"], case["kv_len"]
    if case["form"] not in ("lens", "packed"):
        return [T] * B
    rng = random.Random(B * 100003 + T)
    return [T] + [0 if rng.random() < 0.04 else rng.randint(max(1, T // 10), T) for _ in range(B - 1)]


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    state = {"op": op, "dtype": dt}
    if op in ("norm", "quant"):
        R, C = case["rows"], case["cols"]
        # a residual stream: channels of different sizes, a few of them large
        size = torch.exp(0.5 * torch.randn(C, generator=g, device="cuda"))
        state["x"] = (torch.randn(R, C, generator=g, device="cuda") * size).to(dt)
        if op == "norm":
            state["weight"] = normal(C, std=0.2) + 1.0
            state["residual"] = normal(R, C, std=2.0) if case["residual"] else None
    elif op == "gemm":
        M, K, N = case["rows"], case["k"], case["n"]
        # codes of normal values whose largest of a few thousand stands at 127
        state["act"] = (torch.randn(M, K, generator=g, device="cuda") * 36).round().clamp(-127, 127).to(torch.int8)
        state["wgt"] = (torch.randn(N, K, generator=g, device="cuda") * 36).round().clamp(-127, 127).to(torch.int8)
        state["ascales"] = torch.rand(M, generator=g, device="cuda") * 0.03 + 0.015
        state["wscales"] = (torch.rand(N, generator=g, device="cuda") + 0.5) * (0.028 / math.sqrt(K))
        state["bias"] = normal(N, std=0.1) if case["bias"] else None
    else:
        B, Tq, T, H, Hk, D = (case[k] for k in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))
        form = case["form"]
        lens = torch.tensor(_lengths(case), dtype=torch.int32)
        lens = lens[torch.randperm(B, generator=torch.Generator().manual_seed(seed))]
        state.update(form=form, kv_len=T, kv_lens=None, mask=None, kv_offsets=None)
        # token-major, as the projections leave them
        state["q"] = normal(B, Tq, H, D).transpose(1, 2)
        if form == "packed":
            total = int(lens.sum())
            state["kv_offsets"] = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0).to(torch.int32)]).cuda()
            kv = normal(total, 2, Hk, D)
            state["k"], state["v"] = kv[:, 0], kv[:, 1]
        else:
            kv = normal(B, T, 2, Hk, D)
            state["k"], state["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
            if form == "lens":
                state["kv_lens"] = lens.cuda()
            elif form == "mask":
                state["mask"] = torch.rand(B, T, generator=g, device="cuda") < 0.8
        state["scale"] = D ** -0.5
    return state


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_codes(y):
    """Symmetric 8-bit codes with one scale per row, and that scale."""
    top = y.abs().amax(dim=-1, keepdim=True)
    scale = top / 127.0
    codes = torch.where(top > 0, torch.round(y / scale), torch.zeros_like(y))
    return codes, scale


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + _EPS) * s["weight"].float()
    codes, scale = _plain_codes(y)
    return (codes * scale).to(s["dtype"]), scale[:, 0], (h.to(s["dtype"]) if s["residual"] is not None else None)


def _plain_quant(s):
    codes, scale = _plain_codes(s["x"].float())
    return (codes * scale).to(s["dtype"]), scale[:, 0]


def _plain_gemm(s):
    y = (s["act"].float() @ s["wgt"].float().t()) * s["ascales"][:, None] * s["wscales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["dtype"])


def _plain_cross(s):
    q, k, v, T = s["q"], s["k"], s["v"], s["kv_len"]
    B, H, Tq, D = q.shape
    at = torch.arange(T, device=q.device)
    if s["kv_offsets"] is not None:   # packed -> padded, by index
        off = s["kv_offsets"].long()
        valid = at < (off[1:] - off[:-1])[:, None]
        rows = torch.where(valid, off[:-1, None] + at, 0)
        k, v = k[rows].transpose(1, 2), v[rows].transpose(1, 2)
    elif s["kv_lens"] is not None:
        valid = at < s["kv_lens"][:, None]
    elif s["mask"] is not None:
        valid = s["mask"]
    else:
        valid = None
    group = H // k.shape[1]
    k, v = k.float(), v.float()
    if group > 1:
        k, v = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
    p = (q.float() @ k.transpose(-1, -2)) * s["scale"]
    if valid is not None:
        valid = valid[:, None, None, :]
        p = p.masked_fill(~valid, float("-inf"))
        v = torch.where(valid.transpose(-1, -2), v, torch.zeros((), device=v.device))
        top = p.amax(dim=-1, keepdim=True)
        p = torch.exp(p - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        o = (p @ v) / p.sum(dim=-1, keepdim=True)
        o = torch.where(valid.any(dim=-1, keepdim=True), o, torch.zeros_like(o))
    else:
        p = torch.exp(p - p.amax(dim=-1, keepdim=True))
        o = (p @ v) / p.sum(dim=-1, keepdim=True)
    return o.to(s["dtype"]).transpose(1, 2).reshape(B, Tq, H * D)


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    s, op = state, state["op"]
    if own:
        from nunchaku_b200 import ops

        if op == "norm":
            codes, scales, hidden = ops.rms_norm_quantize_w8a8(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
            return ops.dequantize_w8a8(codes, scales, out_dtype=s["dtype"]), scales, hidden
        if op == "quant":
            codes, scales = ops.quantize_w8a8(s["x"])
            return ops.dequantize_w8a8(codes, scales, out_dtype=s["dtype"]), scales
        if op == "gemm":
            return ops.gemm_w8a8(s["act"], s["wgt"], s["ascales"], s["wscales"], bias=s["bias"], out_dtype=s["dtype"])
        return ops.cross_attention(s["q"], s["k"], s["v"], kv_lens=s["kv_lens"], mask=s["mask"], kv_offsets=s["kv_offsets"],
                                   scale=s["scale"])
    return {"norm": _plain_norm, "quant": _plain_quant, "gemm": _plain_gemm, "cross": _plain_cross}[op](s)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("norm", "quant"):
        n = case["rows"] * case["cols"]
        per = 2 + 1 + (4 if case.get("residual") else 0)          # x, codes (, residual, hidden)
        return {"bytes": n * per + 4 * case["rows"] + (2 * case["cols"] if op == "norm" else 0), "flops": (8 if op == "norm" else 3) * n}
    if op == "gemm":
        M, K, N = case["rows"], case["k"], case["n"]
        return {"bytes": M * K + N * K + 2 * M * N + 4 * M + 4 * N + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    B, Tq, H, Hk, D = (case[k] for k in ("batch", "q_len", "heads", "kv_heads", "dim"))
    states = sum(_lengths(case))
    return {"bytes": 2 * (2 * B * Tq * H * D + 2 * states * Hk * D), "flops": 4 * Tq * states * H * D}


# ---------------------------------------------------------------------------------------------------------------- exact
def _exact_codes(y):
    top = y.abs().max(dim=1).values
    scale = top / 127
    unit = torch.where(top > 0, scale, torch.ones_like(scale))[:, None]
    return torch.round(y / unit) * unit, scale


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("norm", "quant"):
        h = s["x"].double()
        if s["op"] == "quant":
            return _exact_codes(h)
        if s["residual"] is not None:
            h = h + s["residual"].double()
        rms = torch.sqrt(h.square().sum(dim=1) / h.shape[1] + _EPS)
        values, scale = _exact_codes(h / rms[:, None] * s["weight"].double())
        return values, scale, (h if s["residual"] is not None else None)
    if s["op"] == "gemm":
        y = torch.mm(s["act"].double() * s["ascales"].double()[:, None], (s["wgt"].double() * s["wscales"].double()[:, None]).T)
        return y if s["bias"] is None else y + s["bias"].double()
    q = s["q"].double()
    B, H, Tq, D = q.shape
    out = torch.zeros(B, Tq, H, D, dtype=torch.float64, device=q.device)
    bounds = s["kv_offsets"].tolist() if s["kv_offsets"] is not None else None
    lens = s["kv_lens"].tolist() if s["kv_lens"] is not None else None
    for b in range(B):
        if bounds is not None:
            k, v = s["k"][bounds[b]:bounds[b + 1]], s["v"][bounds[b]:bounds[b + 1]]            # [t, Hk, D]
        else:
            k, v = s["k"][b].transpose(0, 1), s["v"][b].transpose(0, 1)
            if lens is not None:
                k, v = k[:lens[b]], v[:lens[b]]
            if s["mask"] is not None:
                k, v = k[s["mask"][b]], v[s["mask"][b]]
        if k.shape[0] == 0:
            continue
        for h in range(H):
            kv = h * k.shape[1] // H
            w = torch.softmax(s["scale"] * (q[b, h] @ k[:, kv].double().T), dim=1)
            out[b, :, h] = w @ v[:, kv].double()
    return out.view(B, Tq, H * D)
