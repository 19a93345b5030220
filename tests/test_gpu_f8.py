"""Linear, gated pair, norm and quantization in 8-bit blocks through the C ABI, against the definitions in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of fp32, relative
U16 = 2.0 ** -11  # of fp16
U8 = 2.0 ** -4    # of e4m3; below 2^-6 its steps are 2^-9
HALF8 = 2.0 ** -10
TINY = 2.0 ** -100
B = 128

E4M3 = np.array([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:119])


@pytest.fixture(scope="module")
def f8():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from helios_glm53flash_amd import f8
    return f8


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def codes(values):
    """float8 tensor of values that e4m3 holds exactly."""
    import torch
    return dev(np.asarray(values, np.float32)).to(torch.float8_e4m3fn)


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def rounded(v):
    """e4m3 of v float64, ties to even (of the codes: entry i has code i)."""
    a = np.abs(v)
    i = np.clip(np.searchsorted(E4M3, a, side="right") - 1, 0, len(E4M3) - 2)
    lo, hi = E4M3[i], E4M3[i + 1]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 1))
    r = np.where(up, hi, lo)
    assert (a[np.isfinite(a)] < 464).all()
    return np.where(np.isnan(v), np.nan, np.copysign(r, v))


def nblocks(k):
    return -(-k // B)


def largest(v):
    """max |v| of the blocks of rows, NaN where one is NaN, at least 2^-100."""
    a = np.stack([np.abs(v[:, b * B:(b + 1) * B]).max(axis=1) for b in range(nblocks(v.shape[1]))], axis=1)
    return np.maximum(a, v.dtype.type(TINY))


def spread(s, K):
    return np.repeat(s, B, axis=1)[:, :K]


def exact_codes(v):
    """Codes' values and scales of fp32 v, by the definition's fp32 operations."""
    with np.errstate(invalid="ignore", over="ignore"):
        a = largest(v)
        f = np.float32(448) / a
        return rounded((v * spread(f, v.shape[1])).astype(np.float64)), a / np.float32(448)


def guarded(shape, dtype, rows=2):
    """An output with rows of a sentinel before and behind it: (whole, view of the output)."""
    import torch
    whole = torch.full((shape[0] + 2 * rows, shape[1]), 7.0, device="cuda").to(dtype)
    return whole, whole[rows:rows + shape[0]]


def check_guard(whole, rows=2):
    w = whole.float()
    assert bool((w[:rows] == 7.0).all()) and bool((w[-rows:] == 7.0).all())


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


# ------------------------------------------------------------------ quantize

QSHAPES = [(1, 16), (1, 128), (3, 144), (1, 4096), (5, 8192), (17, 2048), (33, 1168), (300, 576), (2, 33024), (1, 4194304)]


@pytest.mark.parametrize("ftype", [np.float16, np.float32])
@pytest.mark.parametrize("M,K", QSHAPES)
def test_quantize(f8, M, K, ftype):
    """Bit for bit: the definition is a chain of single fp32 operations."""
    import torch
    r = np.random.default_rng(M + K)
    x = (r.standard_normal((M, K)) * np.exp(r.uniform(-6, 3, (M, nblocks(K)))).repeat(B, axis=1)[:, :K]).astype(ftype)
    x[:, ::97] = 0
    if K >= 384:
        x[0, 128:256] = 0                     # a block of zeros
        x[-1, 256:384] *= ftype(2.0 ** -10)   # steps below the smallest normal code
        x[-1, 300] = 1
    gq, q = guarded((M, K), torch.float8_e4m3fn)
    gs, s = guarded((M, nblocks(K)), torch.float32)
    f8.quantize(dev(x), q, s, M, K)
    want, ws = exact_codes(x.astype(np.float32))
    assert same(s.cpu().numpy(), ws)
    assert same(host(q), want)
    check_guard(gq)
    check_guard(gs)


@pytest.mark.parametrize("ftype", [np.float16, np.float32])
@pytest.mark.parametrize("K,ld,first", [(512, 576, 0), (64, 576, 512), (2048, 12288, 4096), (272, 280, 8)])
def test_quantize_of_strided_rows(f8, K, ld, first, ftype):
    import torch
    M = 9
    x = np.random.default_rng(K).standard_normal((M, ld)).astype(ftype)
    t = dev(x)[:, first:first + K]
    q, s = torch.empty((M, K), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((M, nblocks(K)), device="cuda")
    f8.quantize(t, q, s, M, K)
    want, ws = exact_codes(x[:, first:first + K].astype(np.float32))
    assert same(host(q), want) and same(s.cpu().numpy(), ws)


def test_quantize_keeps_infinities_and_nans_in_their_blocks(f8):
    """What a block with a NaN or an infinity stands for is NaN throughout; the other blocks are as they would be."""
    import torch
    M, K = 6, 400
    x = np.random.default_rng(0).standard_normal((M, K)).astype(np.float16)
    x[0, 5], x[1, 130], x[2, 399], x[3, 256:384], x[4, 0:3] = np.nan, np.inf, -np.inf, -np.inf, (np.inf, np.nan, -np.inf)
    for a in (x, x.astype(np.float32)):
        q, s = torch.empty((M, K), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((M, nblocks(K)), device="cuda")
        f8.quantize(dev(a), q, s, M, K)
        with np.errstate(invalid="ignore"):
            got = host(q) * spread(s.cpu().numpy().astype(np.float64), K)
        bad = spread(np.stack([~np.isfinite(x[:, b * B:(b + 1) * B].astype(float)).all(axis=1) for b in range(nblocks(K))], axis=1), K)
        assert np.isnan(got[bad]).all()
        want, ws = exact_codes(x.astype(np.float32))
        assert same(host(q)[~bad], want[~bad])


@pytest.mark.parametrize("value", [0.0, 2.0 ** -149, 2.0 ** -126, 2.0 ** -101, 2.0 ** -100, 2.0 ** -99, 3.0e38])
def test_quantize_of_the_smallest_and_largest(f8, value):
    import torch
    x = np.full((2, 160), value, np.float32)
    x[1, ::2] *= -1
    q, s = torch.empty((2, 160), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((2, 2), device="cuda")
    f8.quantize(dev(x), q, s, 2, 160)
    want, ws = exact_codes(x)
    assert same(s.cpu().numpy(), ws) and same(host(q), want)


def test_quantize_of_more_rows_than_a_launch_takes(f8):
    import torch
    M, K = (1 << 27) + 7, 16
    x = torch.randn((1 << 20, K), device="cuda").half().repeat((M >> 20) + 1, 1)[:M].contiguous()
    q, s = torch.empty((M, K), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((M, 1), device="cuda")
    f8.quantize(x, q, s, M, K)
    one = torch.empty((1 << 20, K), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((1 << 20, 1), device="cuda")
    f8.quantize(x, *one, 1 << 20, K)
    for at in (0, 64 << 20, 127 << 20, 1 << 27):
        n = min(1 << 20, M - at)
        assert torch.equal(q[at:at + n].view(torch.uint8), one[0][:n].view(torch.uint8)) and torch.equal(s[at:at + n], one[1][:n])


def test_quantize_rounds_ties_to_even(f8):
    """Every halfway value between two codes, and its neighbours in fp32, in a block whose largest value is 448 (factor 1)."""
    import torch
    mid = (E4M3[:-1] + E4M3[1:]) / 2
    v = np.concatenate([mid, np.nextafter(mid.astype(np.float32), np.float32(0)), np.nextafter(mid.astype(np.float32), np.float32(1000)),
                        E4M3]).astype(np.float32)
    v = np.concatenate([v, -v, np.zeros(-2 * len(v) % 127, np.float32)]).reshape(-1, 127)
    x = np.concatenate([v, np.full((len(v), 1), 448, np.float32)], axis=1)
    q, s = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((len(x), 1), device="cuda")
    f8.quantize(dev(x), q, s, len(x), B)
    assert (s.cpu().numpy() == 1).all()
    assert same(host(q), rounded(x.astype(np.float64)))


# ------------------------------------------------------------------ norm

NSHAPES = [(1, 16), (1, 4096), (3, 144), (2, 512), (5, 2048), (4, 4112), (2, 8192), (2, 12288), (3, 16384), (2, 16400), (1, 65536),
           (257, 576)]


def check_norm(h, weight, eps, y=None, q=None, s=None):
    """fp32 sums of squares are off by at most (K + 8) / 2 roundings after the root, the root, quotient and division by K by 4
    more, two products by 2: n is off by at most (K / 2 + 10) 2^-24 relative.  y is rounded once more (2^-11, or half the smallest
    step 2^-25).  The scale's error is n's and one rounding; a code is rounded by half a step of e4m3 (2^-4 relative, or 2^-10)
    after two fp32 roundings."""
    K = h.shape[1]
    n = h / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps) * weight.astype(np.float64)
    rel = (K / 2 + 10) * U32
    if y is not None:
        assert (np.abs(host(y) - n) <= (U16 + 2 * rel) * np.abs(n) + 2.0 ** -25).all()
    if q is not None:
        got_s = s.cpu().numpy().astype(np.float64)
        assert (np.abs(got_s - largest(n) / 448) <= (rel + 2 * U32) * got_s).all()
        ss = spread(got_s, K)
        assert (np.abs(host(q) * ss - n) <= rel * np.abs(n) + (U8 * np.abs(n) + HALF8 * ss) * (1 + 2 * rel + 4 * U32)).all()


@pytest.mark.parametrize("M,K", NSHAPES)
@pytest.mark.parametrize("x32,r32,w32,outs", [(False, False, False, "q"), (True, False, True, "yq"), (False, True, False, "yq"),
                                              (True, True, False, "y"), (False, None, True, "yq"), (True, None, False, "q")])
def test_norm(f8, M, K, x32, r32, w32, outs):
    import torch
    r = np.random.default_rng(M * K)
    x = r.standard_normal((M, K)).astype(np.float32 if x32 else np.float16)
    x[:, 3] *= 30
    w = r.uniform(0.5, 1.5, K).astype(np.float32 if w32 else np.float16)
    res = None if r32 is None else (3 * r.standard_normal((M, K))).astype(np.float32 if r32 else np.float16)
    go, out = guarded((M, K), torch.float32 if r32 else torch.float16) if res is not None else (None, None)
    gy, y = guarded((M, K), torch.float16) if "y" in outs else (None, None)
    gq, q = guarded((M, K), torch.float8_e4m3fn) if "q" in outs else (None, None)
    gs, s = guarded((M, nblocks(K)), torch.float32) if "q" in outs else (None, None)
    eps = 1e-5
    f8.rms_norm(dev(x), dev(w), M, K, eps, None if res is None else dev(res), out, y, q, s)
    h = x.astype(np.float32)
    if res is not None:
        h = (h + res.astype(np.float32)).astype(res.dtype)
        assert same(out.cpu().numpy(), h)
    check_norm(h.astype(np.float64), w, eps, y, q, s)
    for g in (go, gy, gq, gs):
        if g is not None:
            check_guard(g)


def test_norm_in_place_and_of_strided_rows(f8):
    import torch
    M, K = 7, 512
    x = np.random.default_rng(1).standard_normal((M, 576)).astype(np.float16)
    w = np.ones(K, np.float16)
    res = np.random.default_rng(2).standard_normal((M, K)).astype(np.float16)
    t = dev(res)
    y = torch.empty((M, K), dtype=torch.float16, device="cuda")
    f8.rms_norm(dev(x)[:, :K], dev(w), M, K, 1e-6, t, t, y)
    h = (x[:, :K].astype(np.float32) + res.astype(np.float32)).astype(np.float16)
    assert same(t.cpu().numpy(), h)
    check_norm(h.astype(np.float64), w, 1e-6, y)


@pytest.mark.parametrize("K", [256, 16400])
def test_norm_rows_of_zeros_infinities_and_nans(f8, K):
    """Zeros give zeros, also for eps = 0's neighbour; a NaN or infinity stays in its row."""
    import torch
    M = 5
    x = np.random.default_rng(3).standard_normal((M, K)).astype(np.float16)
    x[1] = 0
    x[2, 7], x[3, K - 1] = np.nan, np.inf
    w = np.random.default_rng(4).uniform(0.5, 1.5, K).astype(np.float16)
    y, q, s = (torch.empty((M, K), dtype=torch.float16, device="cuda"), torch.empty((M, K), dtype=torch.float8_e4m3fn, device="cuda"),
               torch.empty((M, nblocks(K)), device="cuda"))
    f8.rms_norm(dev(x), dev(w), M, K, 1e-5, y=y, q=q, scales=s)
    got = host(y)
    assert (got[1] == 0).all() and (host(q)[1] == 0).all()
    assert np.isnan(got[2]).all()
    assert np.isnan(got[3, K - 1]) and (got[3, :K - 1] == 0).all()
    ok = [0, 1, 4]
    check_norm(x[ok].astype(np.float64), w, 1e-5, y[ok], q[ok], s[ok])


def test_norm_of_more_rows_than_a_launch_takes(f8):
    import torch
    M, K = (1 << 21) + 5, 16
    x = torch.randn((M, K), device="cuda").half()
    h, out, w = torch.randn((M, K), device="cuda"), torch.empty((M, K), device="cuda"), torch.rand((K,), device="cuda")
    whole = [torch.empty((M, K), dtype=torch.float16, device="cuda"), torch.empty((M, K), dtype=torch.float8_e4m3fn, device="cuda"),
             torch.empty((M, 1), device="cuda")]
    f8.rms_norm(x, w, M, K, 1e-5, residual=h, out=out, y=whole[0], q=whole[1], scales=whole[2])
    assert torch.equal(out, x.float() + h)
    for a, b in ((0, 1 << 20), (1 << 20, 1 << 21), ((1 << 21) - 3, M)):
        part = [torch.empty_like(t[a:b]) for t in whole]
        f8.rms_norm(x[a:b], w, b - a, K, 1e-5, residual=h[a:b], out=torch.empty_like(out[a:b]), y=part[0], q=part[1], scales=part[2])
        for t, p in zip(whole, part):
            assert torch.equal(t[a:b].view(torch.uint8), p.view(torch.uint8))


# ------------------------------------------------------------------ linear

SHAPES = [  # M, K, N
    (1, 16, 1), (1, 128, 16), (1, 4096, 2048), (1, 144, 33), (2, 4112, 47), (3, 512, 5), (4, 8192, 515), (5, 8192, 260), (7, 1056, 129),
    (8, 4096, 1000), (9, 2048, 96), (16, 4224, 300), (16, 16400, 70), (1, 32016, 40), (6, 20000, 24), (12, 4096, 4096), (17, 656, 200),
    (31, 4096, 130), (33, 96, 64), (45, 4096, 1024), (64, 2080, 257), (65, 1024, 255), (100, 8192, 640), (128, 4096, 384), (129, 352, 129),
    (200, 2048, 1000), (300, 4096, 2304), (513, 1184, 390), (700, 272, 1500), (1025, 512, 640),
]


def weights(f8, seed, N, K, exact):
    """Weights, and their values in float64.  exact: codes are small integers and scales powers of two."""
    r = np.random.default_rng(seed)
    shape = (nblocks(N), nblocks(K))
    c = r.integers(-4, 5, (N, K)).astype(np.float32) if exact else rounded(np.clip(r.standard_normal((N, K)) * 100, -448, 448)).astype(np.float32)
    s = (2.0 ** r.integers(-2, 2, shape) if exact else r.uniform(0.2, 2.0, shape) / (100 * np.sqrt(K))).astype(np.float32)
    return f8.F8Blocks(codes(c), dev(s)), c.astype(np.float64) * spread(np.repeat(s, B, axis=0)[:N].astype(np.float64), K)


def inputs(seed, M, K, exact):
    """Codes and scales on the device, and their values."""
    r = np.random.default_rng(seed)
    c = r.integers(-4, 5, (M, K)).astype(np.float32) if exact else rounded(np.clip(r.standard_normal((M, K)) * 100, -448, 448)).astype(np.float32)
    s = (2.0 ** r.integers(-1, 2, (M, nblocks(K))) if exact else r.uniform(0.002, 0.02, (M, nblocks(K)))).astype(np.float32)
    return codes(c), dev(s), c.astype(np.float64) * spread(s.astype(np.float64), K)


def product_tolerance(x, w):
    """A sum of K products in any order, each block's sum scaled once by a rounded product of scales: at most K + 2 blocks + 2
    roundings of 2^-24, each relative to a partial sum."""
    K = x.shape[1]
    return (K + 2 * nblocks(K) + 2) * U32 * (np.abs(x) @ np.abs(w).T)


def octet_tolerance(x, w):
    """What sums of 8-bit matrix instructions lose, which calls of more than 8 rows with fp16 outputs use: of 8 consecutive k, each product but the one of
    the largest exponent may lose less than 2^-13 of that one's power of two, so 7 * 2^-13 of the largest product at most."""
    import torch
    a, b = torch.from_numpy(np.abs(x)).float().cuda(), torch.from_numpy(np.abs(w)).float().cuda()
    t = torch.zeros((len(x), len(w)), device="cuda")
    for k in range(0, x.shape[1], 8):
        most = a[:, k:k + 1] * b[:, k]
        for j in range(1, 8):
            most = torch.maximum(most, a[:, k + j:k + j + 1] * b[:, k + j])
        t += most
    return 7 * 2.0 ** -13 * 1.001 * host(t)


@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gemm_of_integers_is_exact(f8, M, K, N, fp32):
    """Small integer codes, scales that are powers of two from 2^-3 to 2^2: partial sums are multiples of 1/8 below 2^21, exact in fp32 in any
    order and also where an octet's products are aligned (at most 16, multiples of 1 before the scales), and the fp16 result is the one
    rounding of the exact sum."""
    import torch
    assert K * 16 * 4 < 2 ** 21
    w, w64 = weights(f8, M + K, N, K, True)
    x, xs, x64 = inputs(K + N, M, K, True)
    whole, y = guarded((M, N), torch.float32 if fp32 else torch.float16)
    f8.gemm(y, x, xs, w, M, N, K, fp32)
    torch.cuda.synchronize()
    with np.errstate(over="ignore"):
        want = (x64 @ w64.T).astype(np.float32 if fp32 else np.float16)
    assert np.array_equal(y.cpu().numpy(), want)
    check_guard(whole)


@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("M,K,N", SHAPES[::2] + SHAPES[1:24:2])
def test_gemm_random(f8, M, K, N, fp32):
    import torch
    w, w64 = weights(f8, 3 * M + K, N, K, False)
    x, xs, x64 = inputs(K + 1, M, K, False)
    ref, tol = x64 @ w64.T, product_tolerance(x64, w64)
    if not fp32:
        if M > 8:
            tol = tol + octet_tolerance(x64, w64)
        tol = tol * (1 + U16) + U16 * np.abs(ref) + 2.0 ** -25
    y = torch.empty((M, N), dtype=torch.float32 if fp32 else torch.float16, device="cuda")
    f8.gemm(y, x, xs, w, M, N, K, fp32)
    err = np.abs(host(y) - ref)
    assert (err <= tol).all(), float((err / tol).max())


ALL_M = [1, 2, 4, 5, 8, 9, 16, 17, 20, 33, 64, 65, 70, 129, 260, 513]


@pytest.mark.parametrize("M", ALL_M)
@pytest.mark.parametrize("K", [16, 112, 1120, 2336])
def test_gemm_with_nans_behind_every_edge(f8, M, K):
    """The memory around x, its scales and the weights holds NaN: none of it enters, whatever the tails of M, N and K."""
    import torch
    N = 70
    r = np.random.default_rng(M + K)

    def inside(a, dtype, rows=3):
        whole = torch.full((a.shape[0] + 2 * rows, a.shape[1]), float("nan"), device="cuda").to(dtype)
        whole[rows:-rows] = dev(a.astype(np.float32)).to(dtype)
        return whole[rows:-rows]

    c, wc = r.integers(-4, 5, (M, K)), r.integers(-4, 5, (N, K))
    s, wsc = 2.0 ** r.integers(-1, 2, (M, nblocks(K))), 2.0 ** r.integers(-2, 2, (1, nblocks(K)))
    # rows of scales are 16 bytes apart at most inside; the 8-bit rows keep their 16-byte alignment (K is a multiple of 16)
    x, xs = inside(c, torch.float8_e4m3fn), inside(s, torch.float32)
    w = f8.F8Blocks(inside(wc, torch.float8_e4m3fn), inside(wsc, torch.float32))
    whole, y = guarded((M, N), torch.float32)
    f8.gemm(y, x, xs, w, M, N, K, True)
    want = (c * spread(s, K)) @ (wc * spread(np.repeat(wsc, N, axis=0), K)).T
    assert np.array_equal(host(y), want)
    check_guard(whole)


@pytest.mark.parametrize("M", ALL_M)
def test_gemm_keeps_infinities_and_nans_in_their_rows(f8, M):
    import torch
    K, N = 1056, 300
    w, w64 = weights(f8, 5, N, K, True)
    x, xs, x64 = inputs(6, M, K, True)
    w.codes[7, K - 1] = float("nan")
    w.scales[1, 0] = float("inf")  # the rows 128 .. 255
    rows = np.ones(M, bool)
    if M > 1:
        x[0, 0] = float("nan")
        xs[M - 1, -1] = float("nan")
        rows[[0, M - 1]] = False
    y = torch.empty((M, N), dtype=torch.float32, device="cuda")
    f8.gemm(y, x, xs, w, M, N, K, True)
    got, ref = host(y), x64 @ w64.T
    cols = np.ones(N, bool)
    cols[7] = False
    cols[128:256] = False
    assert np.isnan(got[:, 7]).all() and not np.isfinite(got[:, 128:256]).any()
    if M > 1:
        assert np.isnan(got[0]).all() and np.isnan(got[M - 1]).all()
    assert np.array_equal(got[np.ix_(rows, cols)], ref[np.ix_(rows, cols)])


@pytest.mark.parametrize("M", [1, 8, 16, 45, 300])
def test_gemm_repeats_and_takes_views(f8, M):
    """Two calls give the same bits; weights, inputs and outputs may be views that start inside larger tensors."""
    import torch
    K, N = 2048, 384
    w, w64 = weights(f8, 21, N, K, False)
    x, xs, x64 = inputs(22, M + 3, K, False)
    y = torch.empty((2, M, N), dtype=torch.float32, device="cuda")
    f8.gemm(y[0], x[3:], xs[3:], w, M, N, K, True)
    f8.gemm(y[1], x[3:].clone(), xs[3:].clone(), w, M, N, K, True)
    assert torch.equal(y[0], y[1])
    part = f8.F8Blocks(w.codes[128:], w.scales[1:])
    y2 = torch.empty((M, N - 128), dtype=torch.float32, device="cuda")
    f8.gemm(y2, x[3:], xs[3:], part, M, N - 128, K, True)
    assert (np.abs(host(y2) - host(y[0])[:, 128:]) <= 2 * product_tolerance(x64[3:], w64[128:])).all()


@pytest.mark.parametrize("M", [1, 5, 20, 100, 300])
@pytest.mark.parametrize("N", [1, 3, 17, 130, 131])
def test_gemm_outputs_at_any_alignment(f8, M, N):
    """Rows of y that start at addresses aligned to their type only."""
    import torch
    K = 256
    w, w64 = weights(f8, 31, N, K, True)
    x, xs, x64 = inputs(32, M, K, True)
    for dt in (torch.float32, torch.float16):
        for off in range(4):
            flat = torch.full((M * N + 8,), 7.0, dtype=dt, device="cuda")
            y = flat[off:off + M * N].view(M, N)
            f8.gemm(y, x, xs, w, M, N, K, dt == torch.float32)
            want = (x64 @ w64.T).astype(np.float32 if dt == torch.float32 else np.float16)
            assert np.array_equal(y.cpu().numpy(), want)
            assert bool((flat[:off] == 7).all()) and bool((flat[off + M * N:] == 7).all())


def test_gemm_large_offsets(f8):
    """Codes past 2^32 bytes and outputs past 2^32 elements' bytes: the last rows of a table of 4.3 GB, the last columns of y."""
    import torch
    K, N, M = 4096, 1_060_000, 2100
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("not enough memory")
    c = torch.randint(-4, 5, (1000, K), device="cuda").float().to(torch.float8_e4m3fn)
    w = f8.F8Blocks(c.view(torch.uint8).repeat(N // 1000, 1).view(torch.float8_e4m3fn), torch.ones((nblocks(N), nblocks(K)), device="cuda"))
    x, xs, x64 = inputs(2, M, K, True)
    part = (x64 @ host(c).T).astype(np.float16)
    for m in (1, 16, 40, M):
        y = torch.empty((m, N), dtype=torch.float16, device="cuda")
        f8.gemm(y, x[:m], xs[:m], w, m, N, K)
        for at in (0, N // 2000 * 1000, N - 1000):
            assert np.array_equal(y[:, at:at + 1000].cpu().numpy(), part[:m])
        del y


def test_gemm_of_more_rows_than_a_launch_takes(f8):
    """2^30 rows and some: codes past 2^34 bytes, outputs past 2^34 elements."""
    import torch
    M, K, N = (1 << 30) + 300, 16, 16
    free, _ = torch.cuda.mem_get_info()
    if free < 70 << 30:
        pytest.skip("not enough memory")
    w, w64 = weights(f8, 1, N, K, True)
    some = inputs(2, 1000, K, True)[0]
    x = torch.zeros((M, K), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    xs = torch.ones((M, 1), device="cuda")
    places = [0, (1 << 27) - 500, (1 << 28) - 500, M - 1000]
    for at in places:
        x.view(torch.uint8)[at:at + 1000] = some.view(torch.uint8)
    y = torch.full((M, N), float("nan"), dtype=torch.float16, device="cuda")
    f8.gemm(y, x, xs, w, M, N, K)
    want = (host(some) @ w64.T).astype(np.float16)
    for at in places:
        assert np.array_equal(y[at:at + 1000].cpu().numpy(), want)
        y[at:at + 1000] = 0
    for at in range(0, M, 1 << 27):
        assert not bool(y[at:at + (1 << 27)].any())


# ------------------------------------------------------------------ gated pair

GSHAPES = [  # M, K, N
    (1, 16, 16), (1, 4096, 2048), (2, 144, 48), (3, 1056, 272), (4, 4096, 512), (5, 2048, 1040), (8, 8208, 144), (9, 512, 128),
    (16, 4096, 384), (17, 272, 112), (33, 1024, 640), (45, 4096, 1024), (64, 2048, 272), (100, 4096, 2048), (129, 144, 400), (300, 2048, 1040),
    (513, 512, 256), (1030, 256, 528)]
GWIDE = [(17, 144, 16400), (33, 272, 8208), (45, 528, 12304), (70, 1040, 12304), (20, 4112, 12304), (48, 4112, 8208)]  # many outputs


def gated(x, gw, uw, limit):
    """v and its error: products as in the linear; silu is 1.1-Lipschitz and at most |g|, its exponential is off by (2 |g| + 8) 2^-24."""
    g, u = x @ gw.T, x @ uw.T
    eg, eu = product_tolerance(x, gw), product_tolerance(x, uw)
    g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    with np.errstate(over="ignore"):
        v = g / (1 + np.exp(-g)) * u
    silu = np.abs(v) / np.maximum(np.abs(u), 1e-300)
    return v, 1.1 * eg * (np.abs(u) + eu) + silu * eu + (2 * np.abs(g) + 8) * U32 * np.abs(v)


def check_blocks(q, s, v, ev):
    """Scales: the largest value's error and two roundings; codes half a step of e4m3 after the value's error and two fp32 roundings."""
    got_s = s.cpu().numpy().astype(np.float64)
    K = v.shape[1]
    worst = np.stack([ev[:, b * B:(b + 1) * B].max(axis=1) for b in range(nblocks(K))], axis=1)
    assert (np.abs(got_s - largest(v) / 448) <= worst / 448 + 2 * U32 * got_s).all()
    ss = spread(got_s, K)
    err = np.abs(host(q) * ss - v)
    tol = ev + (U8 * (np.abs(v) + ev) + HALF8 * ss) * (1 + 4 * U32)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("M,K,N,limit", [(*g, limit) for g in GSHAPES for limit in (10.0, 0.5, float("inf"))] + [(*g, 10.0) for g in GWIDE])
def test_gate_up(f8, M, K, N, limit):
    import torch
    gw, gw64 = weights(f8, M + K, N, K, False)
    uw, uw64 = weights(f8, M + K + 1, N, K, False)
    x, xs, x64 = inputs(N, M, K, False)
    gq, q = guarded((M, N), torch.float8_e4m3fn)
    gs, s = guarded((M, nblocks(N)), torch.float32)
    f8.gate_up(q, s, x, xs, gw, uw, M, N, K, limit)
    check_blocks(q, s, *gated(x64, gw64, uw64, limit))
    check_guard(gq)
    check_guard(gs)


@pytest.mark.parametrize("M", ALL_M)
def test_gate_up_nans_and_zeros(f8, M):
    """A NaN in an input row or a weight row makes its blocks NaN and no other; rows of zeros give zeros."""
    import torch
    K, N = 528, 400
    gw, gw64 = weights(f8, 1, N, K, False)
    uw, uw64 = weights(f8, 2, N, K, False)
    x, xs, x64 = inputs(3, M, K, False)
    uw.codes[300, 17] = float("nan")  # block 2
    rows = np.ones(M, bool)
    if M > 2:
        xs[0, 1] = float("nan")
        x[1] = 0
        rows[[0, 1]] = False
    q, s = torch.empty((M, N), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((M, nblocks(N)), device="cuda")
    f8.gate_up(q, s, x, xs, gw, uw, M, N, K)
    v, ev = gated(x64, gw64, uw64, 10.0)
    with np.errstate(invalid="ignore"):
        got = host(q) * spread(s.cpu().numpy().astype(np.float64), N)
    assert np.isnan(got[:, 256:384]).all()
    if M > 2:
        assert np.isnan(got[0]).all()
        assert (got[1, :256] == 0).all() and (got[1, 384:] == 0).all()
    check_blocks(q[rows][:, :256], s[rows][:, :2], v[rows][:, :256], ev[rows][:, :256])
    check_blocks(q[rows][:, 384:], s[rows][:, 3:], v[rows][:, 384:], ev[rows][:, 384:])


@pytest.mark.parametrize("M", ALL_M)
def test_gate_up_with_nans_behind_every_edge(f8, M):
    import torch
    K, N = 144, 176

    def inside(t, rows=3):
        whole = torch.full((t.shape[0] + 2 * rows, t.shape[1]), float("nan"), device="cuda").to(t.dtype)
        whole.view(torch.uint8)[rows:-rows] = t.view(torch.uint8)
        return whole[rows:-rows]

    (gw, gw64), (uw, uw64), (x, xs, x64) = weights(f8, 1, N, K, False), weights(f8, 2, N, K, False), inputs(3, M, K, False)
    gw, uw = f8.F8Blocks(inside(gw.codes), inside(gw.scales)), f8.F8Blocks(inside(uw.codes), inside(uw.scales))
    gq, q = guarded((M, N), torch.float8_e4m3fn)
    gs, s = guarded((M, nblocks(N)), torch.float32)
    f8.gate_up(q, s, inside(x), inside(xs), gw, uw, M, N, K)
    check_blocks(q, s, *gated(x64, gw64, uw64, 10.0))
    check_guard(gq)
    check_guard(gs)


def inside_nans(t, rows=3):
    """A copy of t between rows of NaN."""
    import torch
    whole = torch.full((t.shape[0] + 2 * rows, t.shape[1]), float("nan"), device="cuda").to(t.dtype)
    whole.view(torch.uint8)[rows:-rows] = t.view(torch.uint8)
    return whole[rows:-rows]


LONG_K = [4096, 4112, 4224, 6160, 8192, 12288, 16384, 17408, 17424, 32016]


@pytest.mark.parametrize("M", [1, 3, 8])
@pytest.mark.parametrize("K", LONG_K)
def test_gemm_of_few_long_rows(f8, M, K):
    """As test_gemm_of_integers_is_exact, with NaNs around all inputs."""
    import torch
    N = 72
    assert K * 16 * 4 < 2 ** 21
    w, w64 = weights(f8, M + K, N, K, True)
    x, xs, x64 = inputs(K + 1, M, K, True)
    w, x, xs = f8.F8Blocks(inside_nans(w.codes), inside_nans(w.scales)), inside_nans(x), inside_nans(xs)
    for dt in (torch.float32, torch.float16):
        whole, y = guarded((M, N), dt)
        f8.gemm(y, x, xs, w, M, N, K, dt == torch.float32)
        with np.errstate(over="ignore"):
            want = (x64 @ w64.T).astype(np.float32 if dt == torch.float32 else np.float16)
        assert np.array_equal(y.cpu().numpy(), want)
        check_guard(whole)


@pytest.mark.parametrize("M", [1, 3, 8])
@pytest.mark.parametrize("K", LONG_K)
def test_gate_up_of_few_long_rows(f8, M, K):
    import torch
    N = 144
    (gw, gw64), (uw, uw64), (x, xs, x64) = weights(f8, 1, N, K, False), weights(f8, 2, N, K, False), inputs(3, M, K, False)
    gw, uw = f8.F8Blocks(inside_nans(gw.codes), inside_nans(gw.scales)), f8.F8Blocks(inside_nans(uw.codes), inside_nans(uw.scales))
    gq, q = guarded((M, N), torch.float8_e4m3fn)
    gs, s = guarded((M, nblocks(N)), torch.float32)
    f8.gate_up(q, s, inside_nans(x), inside_nans(xs), gw, uw, M, N, K)
    check_blocks(q, s, *gated(x64, gw64, uw64, 10.0))
    check_guard(gq)
    check_guard(gs)


@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("M", [1, 8, 9, 40, 300])
@pytest.mark.parametrize("K", [384, 400, 4224, 12416])
def test_gemm_of_infinite_scales(f8, M, K, fp32):
    """Positive values and an infinite scale of the last block on either side: what it reaches is not finite (infinity, or NaN where a
    part of the block without values is scaled: K = 400, 0 * infinity), the other rows are as they would be."""
    import torch
    N = 40
    x, w = torch.ones((M, K), device="cuda").to(torch.float8_e4m3fn), torch.ones((N, K), device="cuda").to(torch.float8_e4m3fn)
    xs, ws = torch.ones((M, nblocks(K)), device="cuda"), torch.ones((1, nblocks(K)), device="cuda")
    ys = torch.empty((2, M, N), dtype=torch.float32 if fp32 else torch.float16, device="cuda")
    xs[M // 2, -1] = float("inf")
    f8.gemm(ys[0], x, xs, f8.F8Blocks(w, ws), M, N, K, fp32)
    ws[0, -1] = float("inf")
    f8.gemm(ys[1], x, xs, f8.F8Blocks(w, ws), M, N, K, fp32)
    assert not bool(ys[0, M // 2].isfinite().any()) and not bool(ys[1].isfinite().any())
    ys[0, M // 2] = K
    assert bool((ys[0] == K).all())


@pytest.mark.parametrize("M", [1, 7, 16, 45, 300])
def test_gate_up_repeats(f8, M):
    import torch
    K, N = 2048, 1024
    gw, _ = weights(f8, 1, N, K, False)
    uw, _ = weights(f8, 2, N, K, False)
    x, xs, _ = inputs(3, M, K, False)
    got = []
    for _ in range(3):
        q, s = torch.empty((M, N), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((M, nblocks(N)), device="cuda")
        f8.gate_up(q, s, x, xs, gw, uw, M, N, K)
        got.append((q.view(torch.uint8), s))
    for q, s in got[1:]:
        assert torch.equal(q, got[0][0]) and torch.equal(s, got[0][1])


# ------------------------------------------------------------------ together


def mlp(f8, M, H, N, seed=0):
    """Buffers and calls of norm -> gate and up -> down -> norm over a residual stream, as a layer of a model makes them."""
    import torch
    r = np.random.default_rng(seed)
    t = {"x": dev(r.standard_normal((M, H)).astype(np.float32)), "res": dev(r.standard_normal((M, H)).astype(np.float16)),
         "w": dev(r.uniform(0.5, 1.5, H).astype(np.float16)), "gate": weights(f8, seed + 1, N, H, False), "up": weights(f8, seed + 2, N, H, False),
         "down": weights(f8, seed + 3, H, N, False)}
    e = lambda shape, dt: torch.empty(shape, dtype=dt, device="cuda")  # noqa: E731
    f = torch.float8_e4m3fn
    t |= {"h": e((M, H), torch.float16), "q": e((M, H), f), "s": e((M, nblocks(H)), torch.float32), "q2": e((M, N), f),
          "s2": e((M, nblocks(N)), torch.float32), "d": e((M, H), torch.float32), "h2": e((M, H), torch.float16), "y": e((M, H), torch.float16)}

    def calls(stream=None):
        f8.rms_norm(t["x"], t["w"], M, H, 1e-5, t["res"], t["h"], q=t["q"], scales=t["s"], stream=stream)
        f8.gate_up(t["q2"], t["s2"], t["q"], t["s"], t["gate"][0], t["up"][0], M, N, H, stream=stream)
        f8.gemm(t["d"], t["q2"], t["s2"], t["down"][0], M, H, N, True, stream=stream)
        f8.rms_norm(t["d"], t["w"], M, H, 1e-5, t["h"], t["h2"], y=t["y"], stream=stream)
    return t, calls


def check_mlp(t):
    """Every step against 64 bits on the buffers that it was given."""
    w = t["w"].cpu().numpy()
    values = lambda q, s: host(t[q]) * spread(t[s].cpu().numpy().astype(np.float64), t[q].shape[1])  # noqa: E731
    h = (t["x"].cpu().numpy() + t["res"].cpu().numpy().astype(np.float32)).astype(np.float16)
    assert same(t["h"].cpu().numpy(), h)
    check_norm(h.astype(np.float64), w, 1e-5, q=t["q"], s=t["s"])
    check_blocks(t["q2"], t["s2"], *gated(values("q", "s"), t["gate"][1], t["up"][1], 10.0))
    v = values("q2", "s2")
    assert (np.abs(host(t["d"]) - v @ t["down"][1].T) <= product_tolerance(v, t["down"][1])).all()
    h2 = (t["d"].cpu().numpy() + h.astype(np.float32)).astype(np.float16)
    assert same(t["h2"].cpu().numpy(), h2)
    check_norm(h2.astype(np.float64), w, 1e-5, y=t["y"])


@pytest.mark.parametrize("M", [1, 4, 16, 45, 200])
def test_feed_forward(f8, M):
    t, calls = mlp(f8, M, 1024, 640, seed=M)
    calls()
    check_mlp(t)


@pytest.mark.parametrize("M", [1, 16, 45, 200])
def test_feed_forward_in_a_graph(f8, M):
    """Captured once, replayed with eager calls of the same operators between: every replay equals the eager result."""
    import torch
    t, calls = mlp(f8, M, 2048, 1024, seed=M)
    other, eager = mlp(f8, M + 2, 1024, 640, seed=M + 50)
    keys = ("h", "q", "s", "q2", "s2", "d", "h2", "y")
    raw = lambda k: t[k].view(torch.uint8).clone()  # noqa: E731
    calls()
    want = {k: raw(k) for k in keys}
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        calls()
    for _ in range(4):
        for k in keys:
            t[k].view(torch.uint8).fill_(0x55)
        eager()
        g.replay()
        eager()
        torch.cuda.synchronize()
        for k in keys:
            assert torch.equal(raw(k), want[k]), k
    check_mlp(t)
    check_mlp(other)


def test_calls_on_two_streams_at_once(f8):
    """Streams have workspaces of their own."""
    import torch
    sets = [mlp(f8, M, 2048, 1024, seed=M) for M in (1, 16, 45)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for (_, calls), s in zip(sets, streams):
            calls(s)
    torch.cuda.synchronize()
    for t, _ in sets:
        check_mlp(t)


def test_empty_batches(f8):
    import torch
    w, _ = weights(f8, 1, 32, 128, True)
    f = torch.float8_e4m3fn
    e = lambda shape, dt=torch.float32: torch.empty(shape, dtype=dt, device="cuda")  # noqa: E731
    f8.quantize(e((0, 128)), e((0, 128), f), e((0, 1)), 0, 128)
    f8.rms_norm(e((0, 128)), e((128,)), 0, 128, 1e-5, q=e((0, 128), f), scales=e((0, 1)))
    f8.gemm(e((0, 32)), e((0, 128), f), e((0, 1)), w, 0, 32, 128, True)
    f8.gate_up(e((0, 32), f), e((0, 1)), e((0, 128), f), e((0, 1)), w, w, 0, 32, 128)


def test_python_refusals(f8):
    import torch
    from helios_glm53flash_amd._lib import HxError
    f = torch.float8_e4m3fn
    e = lambda shape, dt=torch.float32: torch.zeros(shape, dtype=dt, device="cuda")  # noqa: E731
    w, _ = weights(f8, 1, 32, 256, True)
    x, xs, y = e((4, 256), f), e((4, 2)), e((4, 32))
    h = torch.float16
    bad = [
        (ValueError, lambda: f8.F8Blocks(e((4, 24), f), e((1, 1)))), (ValueError, lambda: f8.F8Blocks(e((4, 32), f), e((1, 2)))),
        (ValueError, lambda: f8.F8Blocks(e((4, 32)), e((1, 1)))), (ValueError, lambda: f8.F8Blocks(e((4, 32), f), e((1, 1), h))),
        (ValueError, lambda: f8.F8Blocks(e((64, 4), f).t(), e((1, 1)))),
        (ValueError, lambda: f8.gemm(y, x, xs, w, 4, 32, 128, True)), (ValueError, lambda: f8.gemm(y, x, xs, w, 4, 31, 256, True)),
        (ValueError, lambda: f8.gemm(y, x, xs, w, 5, 32, 256, True)), (ValueError, lambda: f8.gemm(y, x, xs[:3], w, 4, 32, 256, True)),
        (ValueError, lambda: f8.gemm(y, x, xs, w, 4, 32, 256, False)), (ValueError, lambda: f8.gemm(y, e((4, 256)), xs, w, 4, 32, 256, True)),
        (ValueError, lambda: f8.gemm(y[:3], x, xs, w, 4, 32, 256, True)), (ValueError, lambda: f8.gemm(y, x, xs, w, -1, 32, 256, True)),
        (HxError, lambda: f8.gemm(x.view(torch.float32).view(-1)[:128].view(4, 32), x, xs, w, 4, 32, 256, True)),
        (ValueError, lambda: f8.gate_up(e((4, 32), f), e((4, 1)), x, xs, w, f8.F8Blocks(e((48, 256), f), e((1, 2))), 4, 32, 256)),
        (ValueError, lambda: f8.gate_up(e((3, 32), f), e((4, 1)), x, xs, w, w, 4, 32, 256)),
        (HxError, lambda: f8.gate_up(e((4, 32), f), e((4, 1)), x, xs, w, w, 4, 32, 256, limit=0.0)),
        (ValueError, lambda: f8.quantize(e((4, 256), torch.bfloat16), x, xs, 4, 256)), (ValueError, lambda: f8.quantize(e((4, 128)), x, xs, 4, 256)),
        (ValueError, lambda: f8.quantize(e((256, 4)).t(), x, xs, 4, 256)), (ValueError, lambda: f8.quantize(e((1, 256)).expand(4, 256), x, xs, 4, 256)),
        (HxError, lambda: f8.quantize(e((4, 260))[:, :256], x, xs, 4, 256)), (HxError, lambda: f8.quantize(e((4, 264))[:, 2:258], x, xs, 4, 256)),
        (HxError, lambda: f8.quantize(e((4, 40)), x, xs, 4, 40)),
        (ValueError, lambda: f8.rms_norm(e((4, 256)), e((255,)), 4, 256, 1e-5, y=e((4, 256), h))),
        (ValueError, lambda: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, residual=e((4, 256)), y=e((4, 256), h))),
        (ValueError, lambda: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, residual=e((4, 256)), out=e((4, 256), h), y=e((4, 256), h))),
        (ValueError, lambda: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, y=e((4, 256), h), q=x)),
        (ValueError, lambda: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, y=e((4, 256)))),
        (HxError, lambda: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5)),
        (HxError, lambda: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, -1.0, y=e((4, 256), h))),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print(i)
    torch.cuda.synchronize()
