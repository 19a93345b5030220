"""Accuracy of the 8-bit linear's sums, and of the norm at its smallest inputs, against the definitions in 64 bits."""
import numpy as np
import pytest

from test_gpu_f8 import E4M3, U16, codes, dev, exact_codes, f8, host, inputs, nblocks, product_tolerance, weights  # noqa: F401

pytestmark = pytest.mark.gpu

SUBNORMAL, NORMAL = E4M3[1:8], E4M3[8:127]


def power(v):
    """2 to the exponent of codes, of those below 2^-6 to -6; 0 of 0."""
    return np.where(v == 0, 0.0, 2.0 ** np.maximum(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -9))), -6))


def octet_loss(x, w):
    """What an octet may lose: its products become multiples of 2^-13 of its largest power of two.  Those with this exponent are such multiples
    (two significands of 3 bits behind the point make 6), so that at most 7 lose, less than one such multiple each."""
    most = np.zeros((len(x), len(w)))
    for k in range(0, x.shape[1], 8):
        t = np.zeros_like(most)
        for j in range(k, k + 8):
            t = np.maximum(t, power(x[:, j])[:, None] * power(w[:, j])[None])
        most += t
    return 7 * 2.0 ** -13 * most


@pytest.mark.parametrize("signs", [False, True])
@pytest.mark.parametrize("kx,kw", [(NORMAL, NORMAL), (NORMAL, SUBNORMAL), (SUBNORMAL, NORMAL), (SUBNORMAL, SUBNORMAL)],
                         ids=["normal", "subnormal_w", "subnormal_x", "subnormal"])
def test_octets_of_unlike_products(f8, kx, kw, signs):
    """fp16 outputs of more than 8 rows: in each octet one product of any codes, normal or not, beside seven of codes up to 1.4.  A second octet
    takes the one away again, so that the outputs are sums of the seven and show what these lost."""
    import torch
    M, N, K, up = 64, 256, 16, 2.0 ** 8
    r = np.random.default_rng(len(kx) + 2 * len(kw) + signs)
    worst = 0.0
    for _ in range(10):
        x, w = np.zeros((M, K)), np.zeros((N, K))
        x[:, 0], w[:, 0] = r.choice(kx, M), r.choice(kw, N)
        x[:, 1:8], w[:, 1:8] = r.choice(E4M3[:60], (M, 7)), r.choice(E4M3[:60], (N, 7))
        if signs:
            x[:, :8] *= r.choice([-1, 1], (M, 8))
            w[:, :8] *= r.choice([-1, 1], (N, 8))
        x[:, 8], w[:, 8] = -x[:, 0], w[:, 0]
        y = torch.empty((M, N), dtype=torch.float16, device="cuda")
        f8.gemm(y, codes(x), torch.full((M, 1), up, device="cuda"), f8.F8Blocks(codes(w), torch.ones((2, 1), device="cuda")), M, N, K)
        ref = up * (x @ w.T)
        tol = product_tolerance(up * x, w) + up * octet_loss(x, w)
        tol = tol * (1 + U16) + U16 * np.abs(ref) + 2.0 ** -25
        worst = max(worst, float((np.abs(host(y) - ref) / tol).max()))
    assert worst <= 1, worst


@pytest.mark.parametrize("M,K,N", [(1, 400, 70), (8, 4224, 200), (9, 2048, 96), (20, 4096, 1024), (45, 8192, 512), (70, 528, 1201), (300, 1040, 640),
                                   (700, 272, 2064)])
def test_exact_products_of_fp16_outputs(f8, M, K, N):
    """exact=True: the fp32 outputs rounded once, bit for bit, whatever M; fp32 outputs are the same with it."""
    import torch
    w, w64 = weights(f8, M, N, K, False)
    x, xs, x64 = inputs(K, M, K, False)
    y32, same32, y16 = torch.empty((M, N), device="cuda"), torch.empty((M, N), device="cuda"), torch.empty((M, N), dtype=torch.float16, device="cuda")
    f8.gemm(y32, x, xs, w, M, N, K, True)
    f8.gemm(same32, x, xs, w, M, N, K, True, exact=True)
    f8.gemm(y16, x, xs, w, M, N, K, exact=True)
    assert (np.abs(host(y32) - x64 @ w64.T) <= product_tolerance(x64, w64)).all()
    assert torch.equal(same32, y32) and torch.equal(y16, y32.half())


def test_exact_products_of_subnormal_codes(f8):
    """Where the cut of 8 consecutive k is coarsest: one product of a subnormal code on one side, 448 on the other, beside smaller ones."""
    import torch
    M, N, K = 16, 32, 16
    x, w = np.full((M, K), 2.0 ** -6), np.full((N, K), 2.0 ** -6)
    x[:, 0], w[:, 0], x[:, 8], w[:, 8] = 448, 2.0 ** -9, -448, 2.0 ** -9
    y = torch.empty((2, M, N), dtype=torch.float16, device="cuda")
    one = torch.ones((M, 1), device="cuda")
    for i in range(2):
        f8.gemm(y[i], codes(x), one, f8.F8Blocks(codes(w), one[:1]), M, N, K, exact=bool(i))
    assert (host(y[1]) == 14 * 2.0 ** -12).all()
    assert (np.abs(host(y[0]) - 14 * 2.0 ** -12) <= octet_loss(x, w) + 2.0 ** -25).all()


@pytest.mark.parametrize("K", [16, 256, 5008, 16400])
def test_norm_at_the_ends_of_its_squares(f8, K):
    """Rows of zeros, of values whose squares are 0 in fp32, and of values whose squares' sum is not finite there, at eps from 0 on; an
    ordinary row beside them is as it would be."""
    import torch
    x = np.repeat(np.float32([0, 2.0 ** -80, 2.0 ** 70, 0.5]), K).reshape(4, K)
    x[1, K // 2:] = 0
    w = np.ones(K, np.float32)
    for eps in (0.0, 2.0 ** -149, 2.0 ** -126, 1e-30, 1e-5):
        y, q, s = (torch.empty((4, K), dtype=torch.float16, device="cuda"), torch.empty((4, K), dtype=torch.float8_e4m3fn, device="cuda"),
                   torch.empty((4, nblocks(K)), device="cuda"))
        f8.rms_norm(dev(x), dev(w), 4, K, eps, y=y, q=q, scales=s)
        got = host(y)
        with np.errstate(invalid="ignore"):
            blocks = host(q) * np.repeat(s.cpu().numpy().astype(np.float64), 128, axis=1)[:, :K]
        if eps == 0:
            assert np.isnan(got[0]).all() and np.isnan(blocks[0]).all()
            assert np.isinf(got[1, :K // 2]).all() and np.isnan(got[1, K // 2:]).all()
        else:
            assert (got[0] == 0).all() and (blocks[0] == 0).all()
            n = 2.0 ** -80 / np.sqrt(eps)  # the squares add nothing to eps
            assert (np.abs(got[1, :K // 2] - n) <= U16 * n + 2.0 ** -24).all() and (got[1, K // 2:] == 0).all()
        assert (got[2] == 0).all() and (blocks[2] == 0).all()
        n = 0.5 / np.sqrt(0.25 + eps)
        assert (np.abs(got[3] - n) <= (U16 + (K + 20) * 2.0 ** -24) * n).all()


def every_code():
    """Values of the 256 codes and a tensor of them."""
    import torch
    c = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    v = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])
    assert np.array_equal(host(c), v, equal_nan=True)
    return v, c


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -12])
@pytest.mark.parametrize("M", [8, 9, 45, 256])
def test_every_code_by_every_code(f8, M, scale):
    """One product an output: exact, and in fp16 rounded once, also to values below its smallest normal one."""
    import torch
    v, c = every_code()
    for k in (0, 7, 8, 77):
        K = 112
        x, w = (torch.zeros((256, K), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
        x[:, k], w[:, k] = c, c
        blocks = f8.F8Blocks(w, torch.full((2, 1), scale, device="cuda"))
        for m in range(0, 256 - M + 1, M):
            with np.errstate(invalid="ignore", over="ignore"):
                want = v[m:m + M, None] * v[None] * scale
                for dt, nt, exact in ((torch.float32, np.float32, False), (torch.float16, np.float16, False), (torch.float16, np.float16, True)):
                    y = torch.empty((M, 256), dtype=dt, device="cuda")
                    f8.gemm(y, x[m:m + M], torch.ones((M, 1), device="cuda"), blocks, M, 256, K, dt == torch.float32, exact=exact)
                    assert np.array_equal(y.cpu().numpy(), want.astype(nt), equal_nan=True)


def test_quantize_of_every_fp16_value(f8):
    """Each of them beside a largest value of every size, bit for bit."""
    import torch
    bits = np.arange(65536, dtype=np.uint16).view(np.float16)
    v = bits[np.isfinite(bits)]
    v = np.concatenate([v, np.zeros(-len(v) % 127, np.float16)]).reshape(-1, 127)
    for top in 2.0 ** np.arange(-24, 16, 3):
        x = np.concatenate([v, np.full((len(v), 1), top, np.float16)], axis=1)
        q, s = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((len(x), 1), device="cuda")
        f8.quantize(dev(x), q, s, len(x), 128)
        want, ws = exact_codes(x.astype(np.float32))
        assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(host(q), want)


@pytest.mark.parametrize("M", [9, 45, 300])
def test_exact_products_in_a_graph(f8, M):
    """Captured with fp32 outputs and 8-bit products beside them, replayed with eager calls between: every replay as the eager result."""
    import torch
    K, N = 4096, 1024
    w, _ = weights(f8, M, N, K, False)
    x, xs, _ = inputs(K, M, K, False)
    ys = [torch.empty((M, N), dtype=t, device="cuda") for t in (torch.float32, torch.float16, torch.float16)]

    def calls():
        f8.gemm(ys[0], x, xs, w, M, N, K, True)
        f8.gemm(ys[1], x, xs, w, M, N, K)
        f8.gemm(ys[2], x, xs, w, M, N, K, exact=True)
    calls()
    want = [y.clone() for y in ys]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        calls()
    for _ in range(4):
        for y in ys:
            y.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, want))
        calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, want))


@pytest.mark.parametrize("M", [8, 200])
def test_gate_over_its_range(f8, M):
    """silu(g) u by its scales, which keep the one value of a block to two roundings: g of either sign from 2^-20 to 100, u = 2^100 |g|, no clamp.
    The exponential, sum, quotient and product are off by (2 |g| + 8) 2^-24, and 0 where the exponential passes fp32's range (its last finite value is
    below exp(88.73)); the scale is rounded twice."""
    import torch
    K, N = 16, 16
    g = np.concatenate([np.geomspace(2.0 ** -20, 100, M - 8), [1, 2, 86, 87, 88, 88.5, 88.9, 99]]).astype(np.float32)[:M]
    for sign in (-1.0, 1.0):
        x, gw, uw = np.zeros((M, K)), np.zeros((N, K)), np.zeros((N, K))
        x[:, 3], gw[:, 3], uw[:, 3] = 1, sign, 1
        one = torch.ones((1, 1), device="cuda")
        q, s = torch.empty((M, N), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((M, 1), device="cuda")
        f8.gate_up(q, s, codes(x), dev(g[:, None]), f8.F8Blocks(codes(gw), one), f8.F8Blocks(codes(uw), 2.0 ** 100 * one), M, N, K, float("inf"))
        g64 = sign * g.astype(np.float64)
        v = np.abs(g64 / (1 + np.exp(-g64)) * g) * 2.0 ** 100
        got = s.cpu().numpy()[:, 0].astype(np.float64)
        want = np.where(g64 < -88.73, 2.0 ** -100, v) / 448
        assert (np.abs(got - want) <= (2 * np.abs(g64) + 10) * 2.0 ** -24 * want).all()
        assert (np.abs(host(q)[:, 0]) == np.where(g64 < -88.73, 0, 448)).all()
