"""Operators around the 4-bit linear and beam search: what a serving engine calls when a model keeps its projections or its
vocabulary head as 4-bit group-scaled words, and when it decodes with several beams.

Kinds of case:
  gemm     ``w4.gemm``: one projection (or the vocabulary head) with 4-bit weights and group scales
  embed    ``w4.embed``: rows of a 4-bit table by token (the head's words used as the embedding), times a scale
  select   ``beam.select``: log-softmax over the vocabulary, plus the beams' scores, the best n over beams and vocabulary
  reorder  ``beam.reorder``: the surviving beams' states copied from their parents

4-bit words: weight (r, k) = scales[r][k / group] * (q - zeros[r][k / group]), zeros 8 where there are none.  A row holds
ceil(K / 128) blocks of 16 int32 words; word 4 g + j of a block holds the 8 weights k = 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7)
of the block in its nibbles, lowest first.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # True: the framework's kernels; False: the plain forms below

NIBBLE_K = (0, 2, 4, 6, 1, 3, 5, 7)
EOS = 2  # the token that a finished beam goes on with


def _gemm(name, M, K, N, group, zeros, fp32):
    return {"name": name, "kind": "gemm", "M": M, "K": K, "N": N, "group": group, "zeros": zeros, "fp32": fp32}


def _embed(name, T, K, N, group, zeros, fp32):
    return {"name": name, "kind": "embed", "T": T, "K": K, "N": N, "group": group, "zeros": zeros, "fp32": fp32}


def _select(name, batch, beams, vocab, n, fp32, done):
    return {"name": name, "kind": "select", "batch": batch, "beams": beams, "vocab": vocab, "n": n, "fp32": fp32, "done": done}


def _reorder(name, layers, batch, beams, out_beams, tokens, max_tokens, width):
    return {"name": name, "kind": "reorder", "layers": layers, "batch": batch, "beams": beams, "out_beams": out_beams,
            "tokens": tokens, "max_tokens": max_tokens, "width": width}


def listed():
    return [
        # the smallest call: one small projection for one token (launch and latency)
        _gemm("w4_m1_small", 1, 4096, 2048, 128, False, True),
        # attention projection of a plain decode step
        _gemm("w4_proj_m1", 1, 4096, 12288, 128, False, False),
        # output projection for the rows of a speculative verify step, fine groups with zero points
        _gemm("w4_o_proj_m5", 5, 8192, 4096, 32, True, False),
        # attention projection for the tokens of a batched decode step
        _gemm("w4_proj_m45", 45, 4096, 12288, 64, True, False),
        # vocabulary head for eight beams
        _gemm("w4_lm_head_m8", 8, 4096, 151552, 128, False, True),
        # a prefill chunk through the widest attention projection; the last tile of rows is ragged
        _gemm("w4_proj_m2000", 2000, 4096, 24576, 128, False, False),
        # the next token's row, and the rows of a prefill chunk
        _embed("embed_1", 1, 4096, 151552, 128, False, False),
        _embed("embed_2000", 2000, 4096, 151552, 64, True, False),
        # one sequence of four beams: the two best continuations of each beam
        _select("select_b1_w4", 1, 4, 151552, 8, True, False),
        # a batch of sequences, eight beams each, some of them finished
        _select("select_b32_w8", 32, 8, 151552, 16, False, True),
        # a small recurrent state of one sequence's beams
        _reorder("reorder_small", 3, 1, 4, 4, 4, 4, 1024),
        # the latent cache of every layer, filled to a ragged length below its capacity
        _reorder("reorder_cache", 42, 4, 8, 8, 1000, 1024, 576),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("gemm", "gemm", "gemm", "embed", "select", "select", "reorder"))
    if kind == "gemm":
        K, N = 32 * _log_uniform(rng, 4, 400), _log_uniform(rng, 64, 40000)
        M = min(_log_uniform(rng, 1, 2048), (2000 * 4096 * 24576) // (K * N))
        case = _gemm("", max(1, M), K, N, rng.choice((32, 64, 128, 128, 256)), rng.random() < 0.5, rng.random() < 0.5)
    elif kind == "embed":
        case = _embed("", _log_uniform(rng, 1, 2000), 32 * _log_uniform(rng, 4, 256), _log_uniform(rng, 100, 151552),
                      rng.choice((32, 64, 128)), rng.random() < 0.5, rng.random() < 0.5)
    elif kind == "select":
        beams = rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
        vocab = _log_uniform(rng, 200, 151552)
        n = rng.randint(1, 2 * beams)
        batch = max(1, min(_log_uniform(rng, 1, 64), 256 // beams, 4096 // (beams * n)))
        case = _select("", batch, beams, vocab, n, rng.random() < 0.5, rng.random() < 0.5)
    else:
        tokens = _log_uniform(rng, 1, 1500)
        beams, batch = rng.randint(1, 12), _log_uniform(rng, 1, 8)
        width = rng.choice((1, 8)) * _log_uniform(rng, 8, 256)
        layers = max(1, min(_log_uniform(rng, 1, 42), 700_000_000 // (batch * beams * tokens * width)))
        case = _reorder("", layers, batch, beams, rng.randint(1, beams + 2), tokens, tokens + rng.choice((0, 1, 40)), width)
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _words(q):
    """int32 words [rows][Kp / 8] of codes q uint8 [rows][Kp], Kp a multiple of 128 (layout at the top)."""
    o = q.view(q.shape[0], -1, 4, 4, 8).transpose(2, 3)  # blocks x (j, g) octets -> blocks x (g, j)
    w = torch.zeros(o.shape[:-1], dtype=torch.int64, device=q.device)
    for i, k in enumerate(NIBBLE_K):
        w |= o[..., k].to(torch.int64) << (4 * i)
    w = torch.where(w >= 1 << 31, w - (1 << 32), w)
    return w.to(torch.int32).reshape(q.shape[0], -1).contiguous()


def _w4_weights(case, g):
    """Codes of a rounded normal distribution about the zero point, scales that give the weights a variance near 1 / K."""
    N, K, group = case["N"], case["K"], case["group"]
    G, Kp = -(-K // group), -(-K // 128) * 128
    zeros = torch.randint(5, 11, (N, G), generator=g, device="cuda").to(torch.uint8) if case["zeros"] else None
    scales = ((0.5 + torch.rand((N, G), generator=g, device="cuda")) * (0.4 / math.sqrt(K))).to(torch.float16)
    words = torch.empty((N, Kp // 8), dtype=torch.int32, device="cuda")
    group_of = (torch.arange(Kp, device="cuda") // group).clamp_(max=G - 1)
    rows = max(1, (1 << 26) // Kp)
    for r in range(0, N, rows):
        q = torch.randn((min(rows, N - r), Kp), generator=g, device="cuda") * 2.5
        q = q + (zeros[r:r + rows].to(torch.float32)[:, group_of] if case["zeros"] else 8)
        q = q.round_().clamp_(0, 15).to(torch.uint8)
        q[:, K:] = 0
        words[r:r + rows] = _words(q)
    return words, scales, zeros


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    dt = torch.float32 if case.get("fp32") else torch.float16
    if case["kind"] in ("gemm", "embed"):
        s["words"], s["scales"], s["zeros"] = _w4_weights(case, g)
        if own:
            from helios_glm53flash_amd import w4
            s["w"] = w4.W4Words(s["words"], s["scales"], s["zeros"], case["K"], case["group"])
        if case["kind"] == "gemm":
            s["x"] = torch.randn((case["M"], case["K"]), generator=g, device="cuda").to(torch.float16)
            s["y"] = torch.empty((case["M"], case["N"]), dtype=dt, device="cuda")
        else:
            s["tokens"] = torch.randint(0, case["N"], (case["T"],), generator=g, device="cuda")
            s["y"] = torch.empty((case["T"], case["K"]), dtype=dt, device="cuda")
    elif case["kind"] == "select":
        rows, V, n = case["batch"] * case["beams"], case["vocab"], case["n"]
        logits = torch.randn((rows, V), generator=g, device="cuda") * 3
        logits[torch.rand((rows, V), generator=g, device="cuda") < 1e-3] = -math.inf  # tokens that the caller forbids
        s["logits"] = logits.to(dt)
        s["cum"] = -8 * torch.rand((rows,), generator=g, device="cuda") - 4
        s["done"] = (torch.rand((rows,), generator=g, device="cuda") < 0.2).to(torch.uint8) if case["done"] else None
        s["scores"] = torch.empty((case["batch"], n), dtype=torch.float32, device="cuda")
        s["parents"] = torch.empty((case["batch"], n), dtype=torch.int64, device="cuda")
        s["tokens"] = torch.empty((case["batch"], n), dtype=torch.int64, device="cuda")
    else:
        b, w, ow = case["batch"], case["beams"], case["out_beams"]
        cache = torch.randn((case["layers"], b * w, case["max_tokens"], case["width"]), dtype=torch.float16, generator=g,
                            device="cuda")
        s["src"] = cache[:, :, :case["tokens"]]
        s["dst"] = torch.zeros((case["layers"], b * ow, case["max_tokens"], case["width"]), dtype=torch.float16,
                               device="cuda")[:, :, :case["tokens"]]
        s["parents"] = torch.randint(0, w, (b, ow), generator=g, device="cuda")
    return s


# ------------------------------------------------------------------ one pass


def _plain_codes(words, K):
    """Codes [rows][K] of words [rows][Kp / 8], float32."""
    shifts = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    nib = (words.unsqueeze(-1) >> shifts) & 15                              # [rows][words][nibble]
    oct_ = nib.view(*words.shape, 2, 4).transpose(-1, -2)                   # nibble 4 h + p holds k = 2 p + h
    blocks = oct_.reshape(words.shape[0], -1, 4, 4, 8).transpose(2, 3)      # word 4 g + j holds octet 4 j + g
    return blocks.reshape(words.shape[0], -1)[:, :K].to(torch.float32)


def _plain_weights(words, scales, zeros, K, group):
    q = _plain_codes(words, K)
    z = zeros.to(torch.float32).repeat_interleave(group, dim=1)[:, :K] if zeros is not None else 8.0
    return (q - z) * scales.to(torch.float32).repeat_interleave(group, dim=1)[:, :K]


def _plain_select(case, logits, cum, done):
    batch, beams, V, n = case["batch"], case["beams"], case["vocab"], case["n"]
    # in 64 bits: candidates of different beams may lie closer than the rounding of 32-bit scores
    x = logits.to(torch.float64)
    top = x.amax(dim=1, keepdim=True)
    lse = (x - top).exp_().sum(dim=1, keepdim=True).log() + top
    score = x - lse + cum.to(torch.float64).unsqueeze(1)
    if done is not None:
        fin = done != 0
        score[fin] = -math.inf
        score[:, EOS] = torch.where(fin, cum.to(torch.float64), score[:, EOS])
    score = torch.where(score.isnan(), -math.inf, score).view(batch, beams * V)
    scores, at = [], []
    for _ in range(n):  # the lowest index among equals each time
        i = score.argmax(dim=1, keepdim=True)
        scores.append(score.gather(1, i))
        at.append(i)
        score.scatter_(1, i, -math.inf)
    scores, at = torch.cat(scores, dim=1), torch.cat(at, dim=1)
    none = scores == -math.inf
    return {"scores": scores.to(torch.float32), "parents": torch.where(none, -1, at // V), "tokens": torch.where(none, -1, at % V)}


def run(s):
    case = s["case"]
    if case["kind"] == "gemm":
        if own:
            from helios_glm53flash_amd import w4
            w4.gemm(s["y"], s["x"], s["w"], case["M"], case["N"], case["K"], case["fp32"])
            return s["y"]
        y = s["x"].to(torch.float32) @ _plain_weights(s["words"], s["scales"], s["zeros"], case["K"], case["group"]).T
        return y.to(s["y"].dtype)
    if case["kind"] == "embed":
        scale = math.sqrt(case["K"])
        if own:
            from helios_glm53flash_amd import w4
            w4.embed(s["w"], s["tokens"], s["y"], case["T"], scale)
            return s["y"]
        t = s["tokens"]
        w = _plain_weights(s["words"][t], s["scales"][t], s["zeros"][t] if s["zeros"] is not None else None, case["K"],
                           case["group"])
        return (w * scale).to(s["y"].dtype)
    if case["kind"] == "select":
        if own:
            from helios_glm53flash_amd import beam
            beam.select(s["logits"], s["cum"], s["done"], s["scores"], s["parents"], s["tokens"], case["batch"],
                        case["beams"], case["vocab"], case["n"], EOS)
            return {k: s[k] for k in ("scores", "parents", "tokens")}
        return _plain_select(case, s["logits"], s["cum"], s["done"])
    if own:
        from helios_glm53flash_amd import beam
        beam.reorder(s["src"], s["parents"], s["dst"], case["batch"], case["beams"], case["out_beams"], dim=1)
        return s["dst"]
    first = torch.arange(case["batch"], device="cuda").unsqueeze(1) * case["beams"]
    return s["src"][:, (first + s["parents"]).view(-1)]


# ------------------------------------------------------------------ work


def _row_bytes(case):
    """Bytes of one row of 4-bit words with its scales and zero points."""
    return case["K"] / 2 + -(-case["K"] // case["group"]) * (3 if case["zeros"] else 2)


def work(case):
    out = 4 if case.get("fp32") else 2
    if case["kind"] == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": N * _row_bytes(case) + 2 * M * K + out * M * N, "flops": 2.0 * M * K * N}
    if case["kind"] == "embed":
        return {"bytes": case["T"] * (_row_bytes(case) + 8 + out * case["K"]), "flops": 2.0 * case["T"] * case["K"]}
    if case["kind"] == "select":
        rows = case["batch"] * case["beams"]
        # per logit: its difference to the maximum, the exponential, the sum
        return {"bytes": rows * (case["vocab"] * out + 5) + case["batch"] * case["n"] * 20, "flops": 3.0 * rows * case["vocab"]}
    copied = 2.0 * case["layers"] * case["batch"] * case["out_beams"] * case["tokens"] * case["width"]
    read = 2.0 * case["layers"] * case["batch"] * min(case["beams"], case["out_beams"]) * case["tokens"] * case["width"]
    return {"bytes": copied + read + 8 * case["batch"] * case["out_beams"], "flops": 0.0}


# ------------------------------------------------------------------ the same in 64 bits


def _exact_parts(case, s, rows):
    """Codes minus zero points [rows][K] and the group of each k, in float64, from the words one nibble at a time."""
    words = s["words"][rows].to(torch.int64) & 0xFFFFFFFF
    K, dev = case["K"], words.device
    k = torch.arange(K, device=dev)
    block, j, g, o = k // 128, k % 128 // 32, k % 32 // 8, k % 8
    nibble = o // 2 + 4 * (o % 2)
    q = (words[:, 16 * block + 4 * g + j] >> (4 * nibble)) & 15
    group = k // case["group"]
    z = s["zeros"][rows].to(torch.int64)[:, group] if s["zeros"] is not None else 8
    return (q - z).to(torch.float64), group


def _exact_select(case, s):
    batch, beams, V, n = case["batch"], case["beams"], case["vocab"], case["n"]
    logits = s["logits"].cpu().numpy()
    cum = s["cum"].cpu().numpy().astype(np.float64)
    done = s["done"].cpu().numpy() if s["done"] is not None else np.zeros(batch * beams, np.uint8)
    scores = np.full((batch, n), -np.inf)
    parents, tokens = np.full((batch, n), -1, np.int64), np.full((batch, n), -1, np.int64)
    for b in range(batch):
        found = []  # (-score, beam, token): the best n of each beam
        for w in range(beams):
            r = b * beams + w
            if done[r]:
                found.append((-cum[r], w, EOS))
                continue
            x = logits[r].astype(np.float64)
            top = x.max()
            if not np.isfinite(top):
                continue
            lse = top + np.log(np.exp(x - top).sum())
            m = min(n, V)
            least = -np.partition(-x, m - 1)[m - 1]
            at = np.flatnonzero(x >= least)
            at = at[np.argsort(-x[at], kind="stable")][:m]
            found += [(-(cum[r] + (x[t] - lse)), w, int(t)) for t in at if x[t] > -np.inf]
        for i, (v, w, t) in enumerate(sorted(f for f in found if f[0] < np.inf)[:n]):
            scores[b, i], parents[b, i], tokens[b, i] = -v, w, t
    return {"scores": torch.from_numpy(scores), "parents": torch.from_numpy(parents), "tokens": torch.from_numpy(tokens)}


def exact(case, seed):
    if case["kind"] == "reorder":  # copies
        return None
    s = prepare(case, seed)
    if case["kind"] == "select":
        return _exact_select(case, s)
    if case["kind"] == "embed":
        d, group = _exact_parts(case, s, s["tokens"])
        return d * s["scales"][s["tokens"]].to(torch.float64)[:, group] * math.sqrt(case["K"])
    x = s["x"].to(torch.float64)
    out = []
    for r in range(0, case["N"], 4096):
        rows = slice(r, min(r + 4096, case["N"]))
        d, group = _exact_parts(case, s, rows)
        out.append(x @ (d * s["scales"][rows].to(torch.float64)[:, group]).T)
    return torch.cat(out, dim=1)
