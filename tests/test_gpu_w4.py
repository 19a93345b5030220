"""Linear and row lookup over 4-bit words with group scales, through the C ABI, against the definition in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of fp32, relative
U16 = 2.0 ** -11  # of fp16


@pytest.fixture(scope="module")
def w4():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from helios_glm53flash_amd import w4
    return w4


def make(seed, N, K, group, zeros, exact=False):
    """Codes, scales and zero points as numpy arrays, and the weights in float64.  exact: scales are powers of two, so that
    sums of integer inputs are exact in fp32."""
    r = np.random.default_rng(seed)
    G = -(-K // group)
    q = r.integers(0, 16, (N, K), dtype=np.uint8)
    s = (2.0 ** r.integers(-2, 2, (N, G)) if exact else r.uniform(0.2, 2.0, (N, G)) / np.sqrt(K)).astype(np.float16)
    z = r.integers(0, 16, (N, G), dtype=np.uint8) if zeros else None
    gi = np.arange(K) // group
    w = s.astype(np.float64)[:, gi] * (q.astype(np.float64) - (z.astype(np.float64)[:, gi] if zeros else 8.0))
    return q, s, z, w


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def words(w4, q, s, z, K, group):
    return w4.W4Words(w4.pack(dev(q)), dev(s), dev(z) if z is not None else None, K, group)


def guarded(shape, dtype, rows=2):
    """An output with rows of a sentinel before and behind it: (whole, view of the output)."""
    import torch
    whole = torch.full((shape[0] + 2 * rows, shape[1]), 77.0, dtype=dtype, device="cuda")
    return whole, whole[rows:rows + shape[0]]


def check_guard(whole, rows=2):
    assert bool((whole[:rows] == 77.0).all()) and bool((whole[-rows:] == 77.0).all())


SHAPES = [  # M, K, N, group, zeros
    (1, 32, 1, 32, False), (1, 128, 16, 128, True), (1, 4096, 2048, 128, False), (1, 160, 33, 32, True),
    (2, 4128, 47, 64, True), (3, 512, 5, 64, False), (4, 8192, 515, 32, True), (5, 8192, 260, 32, True),
    (7, 1056, 129, 256, False), (8, 4096, 1000, 128, True), (9, 2048, 96, 64, False), (16, 4224, 300, 128, True),
    (16, 16416, 70, 128, True), (1, 33024, 40, 256, False), (6, 20000, 24, 64, True),
    (17, 640, 200, 32, True), (31, 4096, 130, 128, False), (33, 96, 64, 64, True), (45, 4096, 1024, 64, True),
    (64, 2080, 257, 128, False), (65, 1024, 255, 32, True), (128, 4096, 384, 128, True), (129, 352, 129, 256, True),
    (200, 2048, 1000, 64, False), (513, 1184, 390, 128, True),
]


@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("M,K,N,group,zeros", SHAPES)
def test_gemm_of_integers_is_exact(w4, M, K, N, group, zeros, fp32):
    """Integer inputs and scales that are powers of two: every product and partial sum is a multiple of 1/4 below 2^22, so
    fp32 sums are exact in any order and the fp16 result is the one rounding of the exact sum."""
    import torch
    q, s, z, w = make(M + K, N, K, group, zeros, exact=True)
    x = np.random.default_rng(K).integers(-4, 5, (M, K)).astype(np.float16)
    ref = x.astype(np.float64) @ w.T
    assert np.abs(x).astype(np.float64).max() * K * 15 * 2 < 2 ** 22
    whole, y = guarded((M, N), torch.float32 if fp32 else torch.float16)
    w4.gemm(y, dev(x), words(w4, q, s, z, K, group), M, N, K, fp32)
    torch.cuda.synchronize()
    with np.errstate(over="ignore"):
        want = ref.astype(np.float32 if fp32 else np.float16)
    assert np.array_equal(y.cpu().numpy(), want)
    check_guard(whole)


@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("M,K,N,group,zeros", SHAPES[::2] + SHAPES[1:16:2])
def test_gemm_random(w4, M, K, N, group, zeros, fp32):
    """Error of a sum of K products in any order with each group's scale applied to its own sum: at most (K + G + 2) roundings of
    2^-24, each relative to a partial sum, so at most (K + G + 2) 2^-24 sum |x w|; fp16 outputs are rounded once more
    (2^-11 of the value, or half the smallest step, 2^-25)."""
    import torch
    q, s, z, w = make(3 * M + K, N, K, group, zeros)
    x = np.random.default_rng(K + 1).standard_normal((M, K)).astype(np.float16)
    x64 = x.astype(np.float64)
    ref = x64 @ w.T
    tol = (K + -(-K // group) + 2) * U32 * (np.abs(x64) @ np.abs(w).T)
    if not fp32:
        tol = tol * (1 + U16) + U16 * np.abs(ref) + 2.0 ** -25
    y = torch.empty((M, N), dtype=torch.float32 if fp32 else torch.float16, device="cuda")
    w4.gemm(y, dev(x), words(w4, q, s, z, K, group), M, N, K, fp32)
    torch.cuda.synchronize()
    err = np.abs(y.cpu().numpy().astype(np.float64) - ref)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("M", [1, 3, 8, 16, 40, 130])
def test_gemm_zero_points_over_the_whole_byte(w4, M):
    """Zero points are bytes: values above 15 (outside what 4 bits hold) enter exactly too."""
    import torch
    K, N, group = 256, 40, 64
    q, s, z, _ = make(5, N, K, group, True, exact=True)
    z = np.random.default_rng(6).integers(0, 256, z.shape, dtype=np.uint8)
    z[0, 0], z[1, 1] = 255, 0
    gi = np.arange(K) // group
    w = s.astype(np.float64)[:, gi] * (q.astype(np.float64) - z.astype(np.float64)[:, gi])
    x = np.random.default_rng(M).integers(-4, 5, (M, K)).astype(np.float16)
    y = torch.empty((M, N), dtype=torch.float32, device="cuda")
    w4.gemm(y, dev(x), words(w4, q, s, z, K, group), M, N, K, True)
    assert np.array_equal(y.cpu().numpy(), (x.astype(np.float64) @ w.T).astype(np.float32))


@pytest.mark.parametrize("M", [1, 4, 6, 16, 20, 70])
def test_gemm_keeps_infinities_and_nans_in_their_rows(w4, M):
    """A NaN or infinity in one input row or one weight row's scale stays in that row and column of y."""
    import torch
    K, N, group = 1056, 37, 32
    q, s, z, w = make(11, N, K, group, True, exact=True)
    x = np.random.default_rng(3).integers(-4, 5, (M, K)).astype(np.float16)
    ref = x.astype(np.float64) @ w.T
    s[5, -1] = np.inf   # the last group of a weight row
    s[9, 0] = np.nan
    bad_row = M - 1
    if M > 1:
        x[bad_row, K - 1] = np.inf
        x[0, 0] = np.nan
    y = torch.empty((M, N), dtype=torch.float32, device="cuda")
    w4.gemm(y, dev(x), words(w4, q, s, z, K, group), M, N, K, True)
    got = y.cpu().numpy()
    cols = np.ones(N, bool)
    cols[[5, 9]] = False
    rows = np.ones(M, bool)
    if M > 1:
        rows[[0, bad_row]] = False
        assert not np.isfinite(got[0]).any()
        d = q[:, K - 1].astype(int) - z[:, (K - 1) // group]
        assert not np.isfinite(got[bad_row][d != 0]).any()
    assert np.array_equal(got[np.ix_(rows, cols)], ref[np.ix_(rows, cols)].astype(np.float32))
    assert not np.isfinite(got[:, 9]).any()


@pytest.mark.parametrize("M", [9, 17, 33, 65, 129])
@pytest.mark.parametrize("K", [1120, 32, 2336])
def test_gemm_single_rows_behind_a_tile(w4, M, K):
    """A last tile of one row, a part of K without a block, and a last block cut short; the memory behind x holds NaN."""
    import torch
    N, group = 70, 32
    q, s, z, w = make(M + K, N, K, group, True, exact=True)
    whole = torch.full((M + 4, K), float("nan"), dtype=torch.float16, device="cuda")
    x = whole[2:-2]
    x.copy_(torch.from_numpy(np.random.default_rng(M).integers(-3, 4, (M, K))))
    guard, y = guarded((M, N), torch.float32)
    w4.gemm(y, x, words(w4, q, s, z, K, group), M, N, K, True)
    assert np.array_equal(y.cpu().numpy().astype(np.float64), x.cpu().numpy().astype(np.float64) @ w.T)
    check_guard(guard)


def test_gemm_empty_batch(w4):
    import torch
    q, s, z, _ = make(1, 16, 128, 64, True)
    w4.gemm(torch.empty((0, 16), device="cuda"), torch.empty((0, 128), dtype=torch.float16, device="cuda"),
            words(w4, q, s, z, 128, 64), 0, 16, 128, True)


@pytest.mark.parametrize("M", [1, 8, 45, 300])
def test_gemm_rows_do_not_depend_on_the_batch(w4, M):
    """Two calls give the same bits, and weight rows and outputs may be views that start inside larger tensors."""
    import torch
    K, N, group = 2048, 320, 64
    q, s, z, _ = make(21, N, K, group, True)
    w = words(w4, q, s, z, K, group)
    x = torch.randn((M + 3, K), device="cuda").half()
    y = torch.empty((2, M, N), dtype=torch.float32, device="cuda")
    w4.gemm(y[0], x[3:], w, M, N, K, True)
    w4.gemm(y[1], x[3:].clone(), w, M, N, K, True)
    assert torch.equal(y[0], y[1])
    part = w4.W4Words(w.words[33:], w.scales[33:], w.zeros[33:], K, group)
    y2 = torch.empty((M, N - 33), dtype=torch.float32, device="cuda")
    w4.gemm(y2, x[3:], part, M, N - 33, K, True)
    # another tile of columns may take another order of sums
    tol = (K + K // group + 2) * U32 * (x[3:].double().abs() @ weights64(w, K).abs().T)
    assert bool(((y2.double() - y[0][:, 33:].double()).abs() <= 2 * tol[:, 33:]).all())


def weights64(w, K):
    import torch
    from helios_glm53flash_amd import w4
    gi = torch.arange(K, device="cuda") // w.group
    d = w4.unpack(w.words, K).double() - (w.zeros.double()[:, gi] if w.zeros is not None else 8.0)
    return d * w.scales.double()[:, gi]


def test_gemm_large_table_offsets(w4):
    """More than 2^32 bytes of words: the last rows of the table."""
    import torch
    K, group = 16384, 128
    N = (1 << 32) // (K // 2) + 70
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    wd = torch.zeros((N, K // 8), dtype=torch.int32, device="cuda")
    wd[-80:] = torch.randint(-2 ** 31, 2 ** 31 - 1, (80, K // 8), generator=gen, device="cuda").to(torch.int32)
    sc = torch.full((N, K // group), 0.5, dtype=torch.float16, device="cuda")
    w = w4.W4Words(wd, sc, None, K, group)
    tail = w4.W4Words(wd[-80:].clone(), sc[-80:].clone(), None, K, group)
    for M in (1, 20):
        x = torch.randint(-3, 4, (M, K), generator=gen, device="cuda").half()
        y = torch.empty((M, N), dtype=torch.float32, device="cuda")
        w4.gemm(y, x, w, M, N, K, True)
        ref = x.double() @ weights64(tail, K).T
        assert torch.equal(y[:, -80:].double(), ref)
        assert torch.equal(y[:, 0].double(), x.double().sum(dim=1) * -4.0)
    out = torch.empty((2, K), dtype=torch.float32, device="cuda")
    w4.embed(w, torch.tensor([N - 1, N - 80], device="cuda"), out, 2)
    assert torch.equal(out.double(), weights64(tail, K)[[79, 0]])


@pytest.mark.parametrize("M", [1, 6, 16, 45, 200])
def test_gemm_graph_replays_on_another_stream(w4, M):
    import torch
    K, N, group = 1024, 300, 128
    q, s, z, _ = make(31, N, K, group, True)
    w = words(w4, q, s, z, K, group)
    x = torch.randn((M, K), device="cuda").half()
    y = torch.empty((M, N), dtype=torch.float32, device="cuda")
    want = torch.empty_like(y)
    w4.gemm(want, x, w, M, N, K, True)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        w4.gemm(y, x, w, M, N, K, True)
    for rep in range(3):
        x.copy_(torch.randn((M, K), device="cuda").half())
        y.fill_(float("nan"))
        g.replay()
        w4.gemm(want, x, w, M, N, K, True)
        torch.cuda.synchronize()
        assert torch.equal(y, want), rep


@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("T,K,N,group,zeros", [(1, 4096, 300, 128, False), (7, 160, 50, 32, True), (33, 2080, 1000, 64, True),
                                              (1000, 512, 17, 256, False)])
def test_embed(w4, T, K, N, group, zeros, fp32):
    """scale * s is rounded once, its product with the integer once: 2 x 2^-24 relative; fp16 outputs once more."""
    import torch
    q, s, z, w = make(T, N, K, group, zeros)
    tok = np.random.default_rng(T).integers(0, N, T)
    tok[0], tok[-1] = N - 1, 0
    scale = float(np.float32(np.sqrt(K)))
    whole, out = guarded((T, K), torch.float32 if fp32 else torch.float16)
    w4.embed(words(w4, q, s, z, K, group), dev(tok), out, T, scale)
    ref = w[tok] * scale
    tol = 2.01 * U32 * np.abs(ref)
    if not fp32:
        tol = tol + U16 * np.abs(ref) * 1.001 + 2.0 ** -25
    assert (np.abs(out.cpu().numpy().astype(np.float64) - ref) <= tol).all()
    check_guard(whole)


@pytest.mark.parametrize("K,N,group,zeros,scale", [(4128, 70, 32, True, 4128 ** 0.5), (1280, 40, 128, False, 1280 ** 0.5), (160, 33, 64, True, 1 / 3),
                                                   (256, 20, 256, True, -1e-3)])
def test_embed_rounds_once(w4, K, N, group, zeros, scale):
    """A weight is exact in fp32 (9 bits times 11), so its product with the scale is rounded once; fp16 outputs once more."""
    import torch
    q, s, z, _ = make(K + N, N, K, group, zeros)
    if zeros:
        z = np.random.default_rng(K).integers(0, 256, z.shape, dtype=np.uint8)
    gi = np.arange(K) // group
    w = s.astype(np.float64)[:, gi] * (q.astype(np.float64) - (z.astype(np.float64)[:, gi] if zeros else 8.0))
    ref = w * np.float64(np.float32(scale))  # 20 bits times 24: exact
    tok = torch.arange(N, device="cuda")
    ww = words(w4, q, s, z if zeros else None, K, group)
    out = torch.empty((N, K), device="cuda")
    w4.embed(ww, tok, out, N, scale)
    assert np.array_equal(out.cpu().numpy(), ref.astype(np.float32))
    half = torch.empty((N, K), dtype=torch.float16, device="cuda")
    w4.embed(ww, tok, half, N, scale)
    err = np.abs(half.cpu().numpy().astype(np.float64) - ref)
    assert (err <= (U16 * (1 + U32) + U32) * np.abs(ref) + 2.0 ** -25).all()


@pytest.mark.parametrize("n,K", [(1_200_000, 32), (540_000, 8192), (140_000_000, 32)])
def test_embed_many_tokens(w4, n, K):
    """Several launches (2^31 words each); an output of more than 2^32 elements."""
    import torch
    q, s, z, w = make(5, 50, K, 32, True, exact=True)
    tok = torch.randint(0, 50, (n,), device="cuda")
    out = torch.full((n, K), 99.0, dtype=torch.float16, device="cuda")
    w4.embed(words(w4, q, s, z, K, 32), tok, out, n)
    table = dev(w.astype(np.float16))
    part = 500_000_000 // K
    for a in range(0, n, part):
        assert torch.equal(out[a:a + part], table[tok[a:a + part]])


def test_gemm_large_batches(w4):
    """Several launches of tiles, an output of more than 2^32 elements, an input of more than 2^31."""
    import torch
    for M, N, K in ((4200, 1 << 20, 32), (70_000, 64, 32768)):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(N)
        wd = torch.randint(-2 ** 31, 2 ** 31 - 1, (N, -(-K // 128) * 16), generator=gen, device="cuda").to(torch.int32)
        w = w4.W4Words(wd, torch.full((N, K // 32), 0.5, dtype=torch.float16, device="cuda"), None, K, 32)
        x = torch.randint(-2, 3, (M, K), generator=gen, device="cuda", dtype=torch.int8).half()
        y = torch.full((M, N), float("nan"), dtype=torch.float16, device="cuda")
        w4.gemm(y, x, w, M, N, K)
        for rows in ([0, 63, 64, M // 2], [4095 % M, 4096 % M, M - 2, M - 1]):
            ref = x[rows].double() @ weights64(w, K).T  # integers and halves: exact but for the output's rounding
            assert torch.equal(y[rows], ref.half())
        assert not bool(y[:, 0].isnan().any()) and not bool(y[:, -1].isnan().any())


@pytest.mark.parametrize("M", [1, 5, 12, 40, 130])
def test_gemm_longest_rows(w4, M):
    """K at its limit; x is nonzero in few places, the row's ends among them, so that the sums are exact."""
    import torch
    K, N, group = 1 << 22, 70, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(M)
    wd = torch.randint(-2 ** 31, 2 ** 31 - 1, (N, K // 8), generator=gen, device="cuda").to(torch.int32)
    w = w4.W4Words(wd, torch.full((N, K // group), 0.5, dtype=torch.float16, device="cuda"), None, K, group)
    x = torch.zeros((M, K), dtype=torch.float16, device="cuda")
    at = torch.randint(0, K, (300,), generator=gen, device="cuda").unique()
    at = torch.cat([at, torch.tensor([0, 1, K - 1, K - 129, K // 2], device="cuda")]).unique()
    x[:, at] = torch.randint(-3, 4, (M, len(at)), generator=gen, device="cuda").half()
    y = torch.empty((M, N), device="cuda")
    w4.gemm(y, x, w, M, N, K, True)
    codes = torch.stack([w4.unpack(wd[n:n + 1], K)[0, at] for n in range(N)]).double()
    assert torch.equal(y.double(), x[:, at].double() @ ((codes - 8) * 0.5).T)


def test_embed_tokens_outside_the_table(w4):
    import torch
    q, s, z, w = make(2, 20, 128, 64, True, exact=True)
    tok = torch.tensor([3, -1, 19, 20, 1 << 40, -(1 << 40), 0], device="cuda")
    out = torch.full((7, 128), 5.0, device="cuda")
    w4.embed(words(w4, q, s, z, 128, 64), tok, out, 7)
    got = out.cpu().numpy()
    assert (got[[1, 3, 4, 5]] == 0).all()
    assert np.array_equal(got[[0, 2, 6]], w[[3, 19, 0]].astype(np.float32))
    w4.embed(words(w4, q, s, z, 128, 64), tok[:0], out[:0], 0)


@pytest.mark.parametrize("M,K,N,group", [(9, 8192, 300, 32), (16, 4224, 64, 128), (32, 16384, 200, 64), (45, 8192, 4096, 64),
                                         (64, 4096, 2048, 128), (100, 4096, 1000, 32), (128, 8192, 4096, 128), (300, 2048, 512, 64)])
def test_gemm_workspaces_through_the_c_entry(w4, M, K, N, group):
    """A workspace of exactly the size asked for, none, and one that is too small: right each time, nothing written behind it and
    its counters left at zero."""
    import ctypes as C
    import torch
    from helios_glm53flash_amd._lib import lib
    q, s, z, w = make(M, N, K, group, True, exact=True)
    ww = words(w4, q, s, z, K, group)
    x = np.random.default_rng(K).integers(-2, 3, (M, K))
    ref = dev(x).double() @ dev(w).T
    xd = dev(x.astype(np.float16))
    need = lib.hx_w4_gemm_workspace_size(M, N, K)
    st = torch.cuda.current_stream().cuda_stream
    for size in {need, 0, max(need - 16, 0)}:
        ws = torch.full((size + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        ws[:min(size, 65536)].zero_()
        for _ in range(3):
            y = torch.full((M, N), float("nan"), device="cuda")
            assert lib.hx_w4_gemm(y.data_ptr(), xd.data_ptr(), C.byref(ww.c()), M, N, K, 1, st, ws.data_ptr() if size else None,
                                  size) == 0
            assert torch.equal(y.double(), ref)
        assert bool((ws[size:] == 0x5A).all()) and bool((ws[:min(size, 65536)] == 0).all())


def test_counts_beyond_32_bits_are_refused(w4):
    import torch
    q, s, z, _ = make(1, 16, 128, 64, True)
    w = words(w4, q, s, z, 128, 64)
    x, y = torch.zeros((1, 128), dtype=torch.float16, device="cuda"), torch.zeros((1, 16), device="cuda")
    for M in (1 << 32, 1 << 31, -1):
        with pytest.raises(ValueError, match="32 bits"):
            w4.gemm(y, x, w, M, 16, 128, True)
        with pytest.raises(ValueError, match="32 bits"):
            w4.embed(w, torch.zeros(1, dtype=torch.int64, device="cuda"), x, M)


def test_another_device_is_refused(w4):
    """The entry points launch on the current device: tensors elsewhere (here the host) are refused."""
    import torch
    q, s, z, _ = make(1, 16, 128, 64, True)
    w = words(w4, q, s, z, 128, 64)
    with pytest.raises(ValueError, match="device"):
        w4.gemm(torch.empty((1, 16)), torch.empty((1, 128), dtype=torch.float16), w, 1, 16, 128, True)


def test_gemm_of_the_same_rows_in_other_batches(w4):
    """Batches on both sides of where another kernel or tile takes over: a row's sums may come in another order, each within the
    bound of test_gemm_random, and the first rows' results lie within two of it."""
    import torch
    K, N, group = 4128, 300, 32
    q, s, z, w = make(51, N, K, group, True)
    ww = words(w4, q, s, z, K, group)
    x = np.random.default_rng(52).standard_normal((130, K)).astype(np.float16)
    x64 = x.astype(np.float64)
    ref = x64 @ w.T
    tol = (K + -(-K // group) + 2) * U32 * (np.abs(x64) @ np.abs(w).T)
    first = None
    for M in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 130):
        y = torch.full((M, N), float("nan"), device="cuda")
        w4.gemm(y, dev(x[:M]), ww, M, N, K, True)
        got = y.cpu().numpy().astype(np.float64)
        assert (np.abs(got - ref[:M]) <= tol[:M]).all(), M
        first = got[0] if first is None else first
        assert (np.abs(got[0] - first) <= 2 * tol[0]).all(), M


def test_tensors_of_another_device_than_the_current_one_are_refused(w4, monkeypatch):
    """With the current device said to be another one, which is all that the checks look at; nothing is launched."""
    import torch
    from helios_glm53flash_amd import beam
    q, s, z, _ = make(1, 16, 128, 64, True)
    w = words(w4, q, s, z, 128, 64)
    x, y = torch.zeros((1, 128), dtype=torch.float16, device="cuda"), torch.full((1, 16), 7.0, device="cuda")
    tok, par = (torch.full((1, 1), 7, dtype=torch.int64, device="cuda") for _ in range(2))
    score = torch.full((1, 1), 7.0, device="cuda")
    here = torch.cuda.current_device()
    monkeypatch.setattr(w4, "_get_device", lambda: here + 1)
    other = f"current device \\(cuda:{here + 1}\\)"
    with pytest.raises(ValueError, match=other):
        w4.gemm(y, x, w, 1, 16, 128, True)
    with pytest.raises(ValueError, match=other):
        w4.embed(w, tok.view(-1), x, 1)
    with pytest.raises(ValueError, match=other):
        beam.select(y, torch.zeros(1, device="cuda"), None, score, par, tok, 1, 1, 16, 1)
    with pytest.raises(ValueError, match=other):
        beam.reorder(x, par, torch.zeros_like(x), 1, 1, 1)
    monkeypatch.undo()
    object.__setattr__(w, "device_index", here + 1)
    for call in (lambda: w4.gemm(y, x, w, 1, 16, 128, True), lambda: w4.embed(w, tok.view(-1), x, 1)):
        with pytest.raises(ValueError, match=f"weights are on cuda:{here + 1}"):
            call()
    torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in (y, tok, par, score))
