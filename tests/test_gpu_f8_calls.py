"""Calls of the 8-bit operators at the edges of what they take: rows past one launch, NaNs around and inside fp16 outputs' inputs, refusals."""
import numpy as np
import pytest

from test_gpu_f8 import (ALL_M, U16, check_blocks, check_guard, f8, gated, guarded, host, inputs, inside_nans,  # noqa: F401
                         product_tolerance, weights)
from test_gpu_f8_tiles import EXACT, LINEAR, name, octet_loss

pytestmark = pytest.mark.gpu


def test_gate_up_of_more_rows_than_a_launch_takes(f8):
    """2^30 rows in one launch, five in another kernel behind it, which needs a workspace of its own layout: codes past 2^34 bytes."""
    import torch
    M, K, N = (1 << 30) + 5, 16, 16
    free, _ = torch.cuda.mem_get_info()
    if free < 70 << 30:
        pytest.skip("not enough memory")
    (gw, gw64), (uw, uw64), (some, ss, x64) = weights(f8, 1, N, K, False), weights(f8, 2, N, K, False), inputs(3, 1000, K, False)
    x, xs = torch.zeros((M, K), dtype=torch.uint8, device="cuda"), torch.ones((M, 1), device="cuda")
    q, s = torch.full((M, N), 0x55, dtype=torch.uint8, device="cuda"), torch.full((M, 1), 7.0, device="cuda")
    places = [0, (1 << 28) - 500, (1 << 29) - 500, M - 1000]
    for at in places:
        x[at:at + 1000], xs[at:at + 1000] = some.view(torch.uint8), ss
    f = torch.float8_e4m3fn
    f8.gate_up(q.view(f), s, x.view(f), xs, gw, uw, M, N, K)
    for at in places:
        check_blocks(q[at:at + 1000].view(f), s[at:at + 1000], *gated(x64, gw64, uw64, 10.0))
        q[at:at + 1000], s[at:at + 1000] = 0, float(np.float32(2.0 ** -100) / np.float32(448))
    for at in range(0, M, 1 << 27):
        assert not bool((q[at:at + (1 << 27)] & 0x7f).any()) and bool((s[at:at + (1 << 27)] == s[0]).all())


# ------------------------------------------------------------------ fp16 outputs: from 9 rows on the products of the 8-bit instruction


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("M", ALL_M)
@pytest.mark.parametrize("K", [16, 112, 1120, 2336])
def test_fp16_outputs_with_nans_behind_every_edge(f8, M, K, exact):
    """Integers as in test_gemm_of_integers_is_exact, in memory between NaNs: none of them enters, whatever the tails of M, N and K."""
    import torch
    N = 70
    w, w64 = weights(f8, M + K, N, K, True)
    x, xs, x64 = inputs(K + 1, M, K, True)
    w = f8.F8Blocks(inside_nans(w.codes), inside_nans(w.scales))
    whole, y = guarded((M, N), torch.float16)
    f8.gemm(y, inside_nans(x), inside_nans(xs), w, M, N, K, exact=exact)
    with np.errstate(over="ignore"):
        assert np.array_equal(y.cpu().numpy(), (x64 @ w64.T).astype(np.float16))
    check_guard(whole)


def check_bad_values(f8, M, K, N, outputs):
    """NaN codes and scales, and infinite scales, stay in their rows and columns."""
    import torch
    w, w64 = weights(f8, 5, N, K, True)
    x, xs, x64 = inputs(6, M, K, True)
    w.codes[7, K - 1] = float("nan")
    w.codes[9, 0] = float("nan")
    w.scales[1, 0] = float("inf")  # the rows 128 .. 255
    rows, cols = np.ones(M, bool), np.ones(N, bool)
    cols[[7, 9]] = False
    cols[128:256] = False
    if M > 4:
        x[0, 0] = float("nan")
        x[2, K - 1] = float("nan")
        xs[M - 1, -1] = float("nan")
        xs[3, 0] = float("inf")
        rows[[0, 2, 3, M - 1]] = False
    whole, y = guarded((M, N), outputs)
    f8.gemm(y, x, xs, w, M, N, K, outputs == torch.float32)
    check_guard(whole)
    with np.errstate(over="ignore"):
        want = (x64 @ w64.T).astype(np.float32 if outputs == torch.float32 else np.float16)
    got = y.cpu().numpy()
    assert np.isnan(got[:, [7, 9]]).all() and not np.isfinite(got[:, 128:256]).any()
    if M > 4:
        assert np.isnan(got[[0, 2, M - 1]]).all() and not np.isfinite(got[3]).any()
    assert np.array_equal(got[np.ix_(rows, cols)], want[np.ix_(rows, cols)])


@pytest.mark.parametrize("M", ALL_M)
@pytest.mark.parametrize("K", [144, 1056])
def test_fp16_outputs_keep_infinities_and_nans_in_their_rows(f8, M, K):
    import torch
    check_bad_values(f8, M, K, 300, torch.float16)


@pytest.mark.parametrize("outputs,tile,parts,size", [a for a in LINEAR if a[3][2] > 256 or a[2] in (1, 4)], ids=name)
def test_every_tile_keeps_infinities_and_nans_in_their_rows(f8, outputs, tile, parts, size):
    import torch
    M, K, N = size
    check_bad_values(f8, M, K, N, torch.float32 if outputs == EXACT else torch.float16)


@pytest.mark.parametrize("M", [1, 8, 9, 16, 45, 300])
def test_fp16_outputs_repeat_and_take_views(f8, M):
    """Two calls give the same bits; weights, inputs and outputs may be views that start inside larger tensors."""
    import torch
    K, N = 2048, 384
    w, w64 = weights(f8, 21, N, K, False)
    x, xs, x64 = inputs(22, M + 3, K, False)
    y = torch.empty((2, M, N), dtype=torch.float16, device="cuda")
    f8.gemm(y[0], x[3:], xs[3:], w, M, N, K)
    f8.gemm(y[1], x[3:].clone(), xs[3:].clone(), w, M, N, K)
    assert torch.equal(y[0], y[1])
    part = f8.F8Blocks(w.codes[128:], w.scales[1:])
    y2 = torch.empty((M, N - 128), dtype=torch.float16, device="cuda")
    f8.gemm(y2, x[3:], xs[3:], part, M, N - 128, K)
    ref = x64[3:] @ w64[128:].T
    tol = product_tolerance(x64[3:], w64[128:]) + octet_loss(x[3:], xs[3:], part)
    assert (np.abs(host(y2) - ref) <= tol * (1 + U16) + U16 * np.abs(ref) + 2.0 ** -25).all()
