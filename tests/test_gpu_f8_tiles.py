"""Every tile kernel of the 8-bit linear and its gated pair, whole and with K in parts, at sizes that are ragged in all extents.
tests/test_f8_plan.py sees to it that the sizes here reach each of them."""
import numpy as np
import pytest

from test_gpu_f8 import (ALL_M, U16, check_blocks, check_guard, f8, gated, guarded, host, inputs, inside_nans, nblocks,  # noqa: F401
                         product_tolerance, spread, weights)
from test_gpu_f8_sums import power

pytestmark = pytest.mark.gpu

FAST, EXACT, GATED = range(3)  # fp16 outputs, fp32 outputs, gated pair
# (outputs, tile, parts of K): M, K, N
TILES = {
    (FAST, "64x32", 1): (9, 272, 136), (FAST, "64x32", 2): (9, 1680, 4405), (FAST, "64x32", 4): (10, 1568, 135), (FAST, "64x32", 7): (9, 4256, 135),
    (FAST, "64x32", 8): (9, 3600, 131),
    (FAST, "64x64", 1): (2756, 528, 133), (FAST, "64x64", 2): (1357, 2208, 137), (FAST, "64x64", 4): (677, 1904, 138),
    (FAST, "64x64", 8): (34, 6944, 1044),
    (FAST, "128x64", 1): (132, 288, 17297), (FAST, "128x64", 2): (35, 3424, 8281), (FAST, "128x64", 4): (33, 11472, 4099),
    (FAST, "128x128", 1): (207, 272, 12861), (FAST, "128x128", 2): (67, 3520, 8493), (FAST, "128x128", 4): (67, 4016, 4259),
    (FAST, "128x128", 8): (68, 7888, 2710),
    (FAST, "256x256", 1): (689, 800, 16644),
    (EXACT, "64x32", 1): (9, 272, 134), (EXACT, "64x32", 2): (9, 1184, 130), (EXACT, "64x32", 4): (10, 1552, 131), (EXACT, "64x32", 7): (9, 3120, 141),
    (EXACT, "64x32", 8): (10, 3616, 136),
    (EXACT, "64x64", 1): (2851, 400, 135), (EXACT, "64x64", 2): (1385, 2224, 139), (EXACT, "64x64", 4): (36, 1552, 2131),
    (EXACT, "64x64", 8): (37, 5952, 2087),
    (EXACT, "128x64", 1): (135, 400, 16547), (EXACT, "128x64", 2): (71, 6304, 12573), (EXACT, "128x64", 4): (66, 8016, 6374),
    (EXACT, "256x256", 1): (1800, 272, 7878),
    (GATED, "64x32", 1): (9, 400, 144), (GATED, "64x32", 2): (10, 800, 144), (GATED, "64x32", 4): (9, 1568, 144), (GATED, "64x32", 7): (9, 3312, 144),
    (GATED, "64x32", 8): (9, 3776, 144),
    (GATED, "64x64", 1): (33, 1248, 4144), (GATED, "64x64", 2): (161, 2208, 688), (GATED, "64x64", 4): (33, 2704, 1040),
    (GATED, "64x64", 7): (35, 6256, 528), (GATED, "64x64", 8): (35, 5648, 544),
    (GATED, "128x64", 1): (2724, 288, 656), (GATED, "128x64", 2): (2699, 6288, 288), (GATED, "128x64", 4): (2058, 8112, 176),
    (GATED, "256x32", 1): (9, 272, 144), (GATED, "256x32", 2): (9, 960, 8432), (GATED, "256x32", 4): (10, 1984, 6240),
    (GATED, "256x32", 8): (10, 11040, 3088),
    (GATED, "256x64", 1): (2723, 272, 288), (GATED, "256x64", 2): (33, 1696, 8400), (GATED, "256x64", 4): (37, 1840, 4144),
    (GATED, "256x64", 8): (35, 9840, 3216),
    (GATED, "256x256", 1): (966, 400, 6176),
}
# Rows of weights that end in the second block of the tile's two.
TILES2 = {(FAST, "256x256", 1): (700, 816, 16600), (EXACT, "256x256", 1): (1790, 528, 7880)}
ALL = [(*key, size) for tiles in (TILES, TILES2) for key, size in tiles.items()]
LINEAR, PAIR = [a for a in ALL if a[0] != GATED], [a for a in ALL if a[0] == GATED]


def name(v):
    return "x".join(map(str, v)) if isinstance(v, tuple) else str(v)


def octet_loss(x, xs, w):
    """octet_loss of test_gpu_f8_sums with the blocks' scales, on the GPU (whose fp32 sums are off by far less than 1.001)."""
    import torch
    K = w.in_features
    ps = [torch.from_numpy(power(host(c)) * spread(s, K)).float().cuda() for c, s in
          ((x, xs.cpu().numpy()), (w.codes, np.repeat(w.scales.cpu().numpy(), 128, axis=0)[:w.out_features]))]
    out = torch.zeros((len(ps[0]), w.out_features), device="cuda")
    for k in range(0, K, 8):
        most = ps[0][:, k:k + 1] * ps[1][:, k]
        for j in range(k + 1, k + 8):
            most = torch.maximum(most, ps[0][:, j:j + 1] * ps[1][:, j])
        out += most
    return 7 * 2.0 ** -13 * 1.001 * host(out)


def product(f8, outputs, x, xs, w, M, N, K):
    import torch
    whole, y = guarded((M, N), torch.float32 if outputs == EXACT else torch.float16)
    f8.gemm(y, x, xs, w, M, N, K, outputs == EXACT)
    torch.cuda.synchronize()
    check_guard(whole)
    return y


@pytest.mark.parametrize("outputs,tile,parts,size", LINEAR, ids=name)
def test_linear_of_integers_is_exact(f8, outputs, tile, parts, size):
    """As test_gemm_of_integers_is_exact, with NaNs around all inputs."""
    M, K, N = size
    assert K * 16 * 4 < 2 ** 21
    w, w64 = weights(f8, M + K, N, K, True)
    x, xs, x64 = inputs(K + N, M, K, True)
    w = f8.F8Blocks(inside_nans(w.codes), inside_nans(w.scales))
    y = product(f8, outputs, inside_nans(x), inside_nans(xs), w, M, N, K)
    with np.errstate(over="ignore"):
        want = (x64 @ w64.T).astype(np.float32 if outputs == EXACT else np.float16)
    assert np.array_equal(y.cpu().numpy(), want)


@pytest.mark.parametrize("outputs,tile,parts,size", LINEAR, ids=name)
def test_linear(f8, outputs, tile, parts, size):
    """Random codes; two calls give the same bits."""
    import torch
    M, K, N = size
    w, w64 = weights(f8, 3 * M + K, N, K, False)
    x, xs, x64 = inputs(K + 1, M, K, False)
    ref, tol = x64 @ w64.T, product_tolerance(x64, w64)
    if outputs == FAST:
        tol = (tol + octet_loss(x, xs, w)) * (1 + U16) + U16 * np.abs(ref) + 2.0 ** -25
    y = product(f8, outputs, x, xs, w, M, N, K)
    err = np.abs(host(y) - ref)
    assert (err <= tol).all(), float((err / tol).max())
    assert torch.equal(product(f8, outputs, x, xs, w, M, N, K), y)


@pytest.mark.parametrize("outputs,tile,parts,size", PAIR, ids=name)
def test_gated_pair(f8, outputs, tile, parts, size):
    """Random codes with NaNs around all inputs; two calls give the same bits."""
    import torch
    M, K, N = size
    (gw, gw64), (uw, uw64), (x, xs, x64) = weights(f8, 1, N, K, False), weights(f8, 2, N, K, False), inputs(3, M, K, False)
    gw, uw = (f8.F8Blocks(inside_nans(w.codes), inside_nans(w.scales)) for w in (gw, uw))
    x, xs = inside_nans(x), inside_nans(xs)
    got = []
    for _ in range(2):
        (gq, q), (gs, s) = guarded((M, N), torch.float8_e4m3fn), guarded((M, nblocks(N)), torch.float32)
        f8.gate_up(q, s, x, xs, gw, uw, M, N, K)
        check_guard(gq)
        check_guard(gs)
        got.append((q, s))
    check_blocks(*got[0], *gated(x64, gw64, uw64, 10.0))
    assert torch.equal(got[0][0].view(torch.uint8), got[1][0].view(torch.uint8)) and torch.equal(got[0][1], got[1][1])


def test_large_offsets_with_scales(f8):
    """Codes past 2^32 bytes under scales that differ from block to block."""
    import torch
    K, N, M = 4112, 1_050_000, 2100
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("not enough memory")
    r = np.random.default_rng(0)
    c = torch.randint(-4, 5, (1000, K), device="cuda").float().to(torch.float8_e4m3fn)
    s = (2.0 ** r.integers(-2, 2, (nblocks(N), nblocks(K)))).astype(np.float32)
    w = f8.F8Blocks(c.view(torch.uint8).repeat(N // 1000, 1).view(torch.float8_e4m3fn), torch.from_numpy(s).cuda())
    x, xs, x64 = inputs(2, M, K, True)
    c64 = host(c)
    for m in (1, 16, 40, M):
        y = torch.empty((m, N), dtype=torch.float16, device="cuda")
        f8.gemm(y, x[:m], xs[:m], w, m, N, K)
        for at in (0, N // 2000 * 1000, N - 1000):
            scales = spread(s[(np.arange(at, at + 1000)) // 128].astype(np.float64), K)
            with np.errstate(over="ignore"):
                want = (x64[:m] @ (c64 * scales).T).astype(np.float16)
            assert np.array_equal(y[:, at:at + 1000].cpu().numpy(), want)
        del y
