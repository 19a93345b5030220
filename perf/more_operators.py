"""Linears in 8-bit floating point (e4m3) with a scale for each block of 128, and what feeds them: what a serving engine calls for
the projections, the dense layers and the vocabulary head of a model that is stored that way.

Kinds of case:
  gemm      ``f8.gemm``: one projection, inputs and weights in 8 bits
  gate_up   ``f8.gate_up``: gate and up projections, the clamped SiLU gate and the product, output in 8 bits for the down projection
  norm      ``f8.rms_norm``: the residual's addition, the root-mean-square norm and its output in 8 bits and / or fp16
  quantize  ``f8.quantize``: activations that come from elsewhere (an attention output) in 8 bits

Blocks: input rows have a scale for each 128 consecutive k, weights one for each 128 x 128; the last ones may be short.
    a = max(largest |v| of the block, 2^-100)        scale = a / 448        code = e4m3(v * (448 / a)), to nearest even
"""
from __future__ import annotations

import math

import torch

own = False  # True: the framework's kernels; False: the plain forms below

B = 128           # values of a block
TOP = 448.0       # the largest e4m3 value
TINY = 2.0 ** -100
LIMIT = 10.0      # clamp of the gate's inputs
EPS = 1e-5
F8 = torch.float8_e4m3fn


def _gemm(name, M, K, N, fp32):
    return {"name": name, "kind": "gemm", "M": M, "K": K, "N": N, "fp32": fp32}


def _gate_up(name, M, K, N):
    return {"name": name, "kind": "gate_up", "M": M, "K": K, "N": N}


def _norm(name, M, K, x32, residual, r32, y, q):
    return {"name": name, "kind": "norm", "M": M, "K": K, "x32": x32, "residual": residual, "r32": r32, "y": y, "q": q}


def _quantize(name, M, K, x32, ld):
    return {"name": name, "kind": "quantize", "M": M, "K": K, "x32": x32, "ld": ld}


def listed():
    return [
        # the smallest product: one projection for one token (launch and latency)
        _gemm("f8_m1_small", 1, 4096, 2048, True),
        # attention projection of a plain decode step
        _gemm("f8_proj_m1", 1, 4096, 12288, False),
        # vocabulary head for the rows of a batched or speculative step
        _gemm("f8_lm_head_m8", 8, 4096, 151552, True),
        # output projection for the tokens of a batched decode step; the last tile of rows is ragged
        _gemm("f8_o_proj_m45", 45, 8192, 4096, False),
        # a prefill chunk through the widest attention projection
        _gemm("f8_proj_m2000", 2000, 4096, 24576, False),
        # the shared expert of one token
        _gate_up("gate_up_m1", 1, 4096, 2048),
        # the dense layers of a batched decode step
        _gate_up("gate_up_m45", 45, 4096, 12288),
        # and of a prefill chunk
        _gate_up("gate_up_m2000", 2000, 4096, 12288),
        # ahead of a projection, one token
        _norm("norm_1", 1, 4096, False, True, False, False, True),
        # ahead of a router (fp16) and of the experts (8 bits), a prefill chunk; the branch's output comes in fp32
        _norm("norm_2000", 2000, 4096, True, True, False, True, True),
        # attention outputs ahead of the output projection: a speculative step, a prefill chunk as a part of wider rows
        _quantize("quantize_5", 5, 8192, False, 8192),
        _quantize("quantize_2000", 2000, 8192, False, 12288),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("gemm", "gemm", "gemm", "gate_up", "gate_up", "norm", "quantize"))
    most = 2000 * 4096 * 24576
    if kind == "gemm":
        K, N = 16 * _log_uniform(rng, 8, 700), _log_uniform(rng, 64, 40000)
        case = _gemm("", max(1, min(_log_uniform(rng, 1, 2048), most // (K * N))), K, N, rng.random() < 0.5)
    elif kind == "gate_up":
        K, N = 16 * _log_uniform(rng, 8, 512), 16 * _log_uniform(rng, 4, 900)
        case = _gate_up("", max(1, min(_log_uniform(rng, 1, 2048), most // (2 * K * N))), K, N)
    elif kind == "norm":
        y, q = rng.choice(((False, True), (True, True), (True, False)))
        case = _norm("", _log_uniform(rng, 1, 4096), 16 * _log_uniform(rng, 8, 1024), rng.random() < 0.3, rng.random() < 0.8,
                     rng.random() < 0.3, y, q)
    else:
        K = 16 * _log_uniform(rng, 8, 1024)
        case = _quantize("", _log_uniform(rng, 1, 4096), K, rng.random() < 0.3, K + rng.choice((0, 0, 16, 576)))
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _spread(s, K):
    """Scales of blocks [..][ceil(K / 128)] as one per k."""
    return s.repeat_interleave(B, dim=-1)[..., :K]


def _blocks_of(v):
    """v [M][K] as [M][blocks][128], zeros behind K."""
    M, K = v.shape
    return torch.nn.functional.pad(v, (0, -K % B)).view(M, -1, B)


def _to_blocks(v):
    """(codes e4m3 [M][K], scales [M][ceil(K / 128)]) of v fp32 [M][K]."""
    a = _blocks_of(v).abs().amax(dim=2).clamp(min=TINY)
    return (v * _spread(TOP / a, v.shape[1])).to(F8), a / TOP


def _weights(N, K, g):
    """Codes and scales of a normal distribution of variance near 1 / K whose size differs from block to block."""
    nb, kb = -(-N // B), -(-K // B)
    codes = torch.empty((N, K), dtype=F8, device="cuda")
    scales = torch.empty((nb, kb), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // (B * K)) * B
    for r in range(0, N, step):
        n = min(step, N - r)
        rows = -(-n // B)
        size = (0.5 + torch.rand((rows, kb), generator=g, device="cuda")) / math.sqrt(K)
        w = torch.randn((n, K), generator=g, device="cuda") * _spread(size.repeat_interleave(B, dim=0)[:n], K)
        a = torch.nn.functional.pad(w, (0, kb * B - K, 0, rows * B - n)).view(rows, B, kb, B).abs().amax(dim=(1, 3)).clamp(min=TINY)
        codes[r:r + n] = (w * _spread((TOP / a).repeat_interleave(B, dim=0)[:n], K)).to(F8)
        scales[r // B:r // B + rows] = a / TOP
    return codes, scales


def _activations(M, K, g):
    """Rows of different size, some values of a row far above the others, as a residual stream has them."""
    x = torch.randn((M, K), generator=g, device="cuda") * (0.5 + 2 * torch.rand((M, 1), generator=g, device="cuda"))
    return torch.where(torch.rand((M, K), generator=g, device="cuda") < 2e-3, 20 * x, x)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    M, K = case["M"], case["K"]
    empty = lambda shape, dt: torch.empty(shape, dtype=dt, device="cuda")  # noqa: E731
    if case["kind"] in ("gemm", "gate_up"):
        N = case["N"]
        s["x"], s["xs"] = _to_blocks(_activations(M, K, g))
        s["w"] = [_weights(N, K, g) for _ in range(2 if case["kind"] == "gate_up" else 1)]
        if own:
            from helios_glm53flash_amd import f8
            s["blocks"] = [f8.F8Blocks(*w) for w in s["w"]]
        if case["kind"] == "gemm":
            s["y"] = empty((M, N), torch.float32 if case["fp32"] else torch.float16)
        else:
            s["q"], s["scales"] = empty((M, N), F8), empty((M, -(-N // B)), torch.float32)
    elif case["kind"] == "norm":
        s["x"] = _activations(M, K, g).to(torch.float32 if case["x32"] else torch.float16)
        s["weight"] = (0.5 + torch.rand((K,), generator=g, device="cuda")).to(torch.float16)
        s["residual"] = s["h"] = s["y"] = s["q"] = s["scales"] = None
        if case["residual"]:
            s["residual"] = (3 * _activations(M, K, g)).to(torch.float32 if case["r32"] else torch.float16)
            s["h"] = torch.empty_like(s["residual"])
        if case["y"]:
            s["y"] = empty((M, K), torch.float16)
        if case["q"]:
            s["q"], s["scales"] = empty((M, K), F8), empty((M, -(-K // B)), torch.float32)
    else:
        s["x"] = _activations(M, case["ld"], g).to(torch.float32 if case["x32"] else torch.float16)[:, :K]
        s["q"], s["scales"] = empty((M, K), F8), empty((M, -(-K // B)), torch.float32)
    return s


# ------------------------------------------------------------------ one pass


def _product(x, xs, w, ws):
    """fp32 x W^T of dequantized blocks."""
    N, K = w.shape
    wd = w.to(torch.float32) * _spread(ws.repeat_interleave(B, dim=0)[:N], K)
    return (x.to(torch.float32) * _spread(xs, K)) @ wd.T


def _gated(g, u):
    g, u = g.clamp(max=LIMIT), u.clamp(min=-LIMIT, max=LIMIT)
    return g / (1 + (-g).exp()) * u


def run(s):
    case = s["case"]
    M, K = case["M"], case["K"]
    if own:
        from helios_glm53flash_amd import f8
        if case["kind"] == "gemm":
            f8.gemm(s["y"], s["x"], s["xs"], s["blocks"][0], M, case["N"], K, case["fp32"])
            return s["y"]
        if case["kind"] == "gate_up":
            f8.gate_up(s["q"], s["scales"], s["x"], s["xs"], s["blocks"][0], s["blocks"][1], M, case["N"], K, LIMIT)
            return {"q": s["q"], "scales": s["scales"]}
        if case["kind"] == "norm":
            f8.rms_norm(s["x"], s["weight"], M, K, EPS, residual=s["residual"], out=s["h"], y=s["y"], q=s["q"], scales=s["scales"])
            return {"h": s["h"], "y": s["y"], "q": s["q"], "scales": s["scales"]}
        f8.quantize(s["x"], s["q"], s["scales"], M, K)
        return {"q": s["q"], "scales": s["scales"]}
    if case["kind"] == "gemm":
        return _product(s["x"], s["xs"], *s["w"][0]).to(s["y"].dtype)
    if case["kind"] == "gate_up":
        q, scales = _to_blocks(_gated(_product(s["x"], s["xs"], *s["w"][0]), _product(s["x"], s["xs"], *s["w"][1])))
        return {"q": q, "scales": scales}
    if case["kind"] == "quantize":
        q, scales = _to_blocks(s["x"].to(torch.float32))
        return {"q": q, "scales": scales}
    h, out = s["x"].to(torch.float32), None
    if case["residual"]:
        out = (h + s["residual"].to(torch.float32)).to(s["residual"].dtype)
        h = out.to(torch.float32)
    n = h / (h.square().mean(dim=1, keepdim=True) + EPS).sqrt() * s["weight"].to(torch.float32)
    q, scales = _to_blocks(n) if case["q"] else (None, None)
    return {"h": out, "y": n.to(torch.float16) if case["y"] else None, "q": q, "scales": scales}


# ------------------------------------------------------------------ work


def work(case):
    M, K = case["M"], case["K"]
    kb = -(-K // B)
    if case["kind"] in ("gemm", "gate_up"):
        N, n = case["N"], 2 if case["kind"] == "gate_up" else 1
        nb = -(-N // B)
        out = (4 if case["fp32"] else 2) * M * N if n == 1 else M * (N + 4 * nb)
        return {"bytes": n * (N * K + 4 * nb * kb) + M * (K + 4 * kb) + out, "flops": 2.0 * n * M * K * N}
    x = 4 if case["x32"] else 2
    if case["kind"] == "quantize":
        # per value: its size against the largest, the product with the factor
        return {"bytes": M * (x * K + K + 4 * kb), "flops": 2.0 * M * K}
    r = (8 if case["r32"] else 4) if case["residual"] else 0
    out = (2 * K if case["y"] else 0) + (K + 4 * kb if case["q"] else 0)
    # per value: the sum, its square, two products, and where 8 bits are asked for two more
    return {"bytes": M * ((x + r) * K + out) + 2 * K, "flops": (7.0 if case["q"] else 5.0) * M * K}


# ------------------------------------------------------------------ the same in 64 bits


def _exact_product(s, which):
    x, xs = s["x"].to(torch.float64), s["xs"].to(torch.float64)
    (M, K), (w, ws) = x.shape, s["w"][which]
    block = torch.arange(K, device=x.device) // B
    x = x * xs[:, block]
    out = []
    for r in range(0, w.shape[0], 32 * B):
        c = w[r:r + 32 * B].to(torch.float64)
        n = torch.arange(r, r + c.shape[0], device=x.device) // B
        out.append(x @ (c * ws.to(torch.float64)[n][:, block]).T)
    return torch.cat(out, dim=1)


def _exact_blocks(v):
    """Codes before their rounding, and scales."""
    a = torch.stack([p.abs().amax(dim=1) for p in v.split(B, dim=1)], dim=1).clamp_(min=TINY)
    return v * (TOP / a)[:, torch.arange(v.shape[1], device=v.device) // B], a / TOP


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gemm":
        return _exact_product(s, 0)
    if case["kind"] == "gate_up":
        g, u = _exact_product(s, 0).clamp_(max=LIMIT), _exact_product(s, 1).clamp_(-LIMIT, LIMIT)
        v = g * torch.sigmoid(g) * u
    else:
        v = s["x"].to(torch.float64)
    out = {}
    if case["kind"] == "norm":
        out = {"h": None, "y": None, "q": None, "scales": None}
        if case["residual"]:
            v = v + s["residual"].to(torch.float64)
            out["h"] = v
            v = v.to(s["residual"].dtype).to(torch.float64)  # what is normalized is the sum as it is kept
        v = v * (v.square().sum(dim=1, keepdim=True) / case["K"] + EPS).rsqrt() * s["weight"].to(torch.float64)
        if case["y"]:
            out["y"] = v
        if not case["q"]:
            return out
    out["q"], out["scales"] = _exact_blocks(v)
    return out
