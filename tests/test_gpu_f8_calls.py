"""Calls of the 8-bit operators at the edges of what they take: rows past one launch, NaNs around and inside fp16 outputs' inputs, refusals."""
import numpy as np
import pytest
import torch

from helios_glm53flash_amd._lib import HxError

from test_gpu_f8 import (ALL_M, U16, check_blocks, check_guard, f8, gated, guarded, host, inputs, inside_nans, nblocks,  # noqa: F401
                         product_tolerance, weights)
from test_gpu_f8_tiles import EXACT, LINEAR, name, octet_loss

pytestmark = pytest.mark.gpu


def test_gate_up_of_more_rows_than_a_launch_takes(f8):
    """2^30 rows in one launch, five in another kernel behind it, which needs a workspace of its own layout: codes past 2^34 bytes."""
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
    check_bad_values(f8, M, K, 300, torch.float16)


@pytest.mark.parametrize("outputs,tile,parts,size", [a for a in LINEAR if a[3][2] > 256 or a[2] in (1, 4)], ids=name)
def test_every_tile_keeps_infinities_and_nans_in_their_rows(f8, outputs, tile, parts, size):
    M, K, N = size
    check_bad_values(f8, M, K, N, torch.float32 if outputs == EXACT else torch.float16)


@pytest.mark.parametrize("M", [1, 8, 9, 16, 45, 300])
def test_fp16_outputs_repeat_and_take_views(f8, M):
    """Two calls give the same bits; weights, inputs and outputs may be views that start inside larger tensors."""
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


# ------------------------------------------------------------------ refusals, each by itself


F, H = torch.float8_e4m3fn, torch.float16


def blocks(f8, e, N=32, K=256):
    return f8.F8Blocks(e((N, K), F), e((nblocks(N), nblocks(K))))


def gemm_over(f8, x, e):
    f8.gemm(x.view(torch.float32).view(-1)[:128].view(4, 32), x, e((4, 2)), blocks(f8, e), 4, 32, 256, True)


REFUSALS = {  # name: (raised, its text, call of f8 and a maker of zeros)
    "blocks_of_short_k": (ValueError, "multiple of 16", lambda f8, e: f8.F8Blocks(e((4, 24), F), e((1, 1)))),
    "blocks_with_scales_of_another_shape": (ValueError, "scales must be", lambda f8, e: f8.F8Blocks(e((4, 32), F), e((1, 2)))),
    "blocks_of_fp32": (ValueError, "codes", lambda f8, e: f8.F8Blocks(e((4, 32)), e((1, 1)))),
    "blocks_with_fp16_scales": (ValueError, "scales", lambda f8, e: f8.F8Blocks(e((4, 32), F), e((1, 1), H))),
    "blocks_of_columns": (ValueError, "codes", lambda f8, e: f8.F8Blocks(e((64, 4), F).t(), e((1, 1)))),
    "blocks_without_rows": (ValueError, "multiple of 16", lambda f8, e: f8.F8Blocks(e((0, 32), F), e((0, 1)))),
    "gemm_of_another_k": (ValueError, "do not match", lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((4, 2)), blocks(f8, e), 4, 32, 128, True)),
    "gemm_of_another_n": (ValueError, "do not match", lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((4, 2)), blocks(f8, e), 4, 31, 256, True)),
    "gemm_of_too_many_rows": (ValueError, "codes / scales smaller",
        lambda f8, e: f8.gemm(e((5, 32)), e((4, 256), F), e((5, 2)), blocks(f8, e), 5, 32, 256, True)),
    "gemm_of_few_scales": (ValueError, "codes / scales smaller",
        lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((3, 2)), blocks(f8, e), 4, 32, 256, True)),
    "gemm_into_the_other_type": (ValueError, "y", lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((4, 2)), blocks(f8, e), 4, 32, 256)),
    "exact_gemm_into_the_other_type": (ValueError, "y",
        lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((4, 2)), blocks(f8, e), 4, 32, 256, exact=True)),
    "gemm_of_fp32": (ValueError, "dtype", lambda f8, e: f8.gemm(e((4, 32)), e((4, 256)), e((4, 2)), blocks(f8, e), 4, 32, 256, True)),
    "gemm_into_few_rows": (ValueError, "y smaller", lambda f8, e: f8.gemm(e((3, 32)), e((4, 256), F), e((4, 2)), blocks(f8, e), 4, 32, 256, True)),
    "gemm_of_negative_rows": (ValueError, "32 bits", lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((4, 2)), blocks(f8, e), -1, 32, 256, True)),
    "gemm_over_its_input": (HxError, "overlap", lambda f8, e: gemm_over(f8, e((4, 256), F), e)),
    "pair_of_unlike_weights": (ValueError, "do not match",
        lambda f8, e: f8.gate_up(e((4, 32), F), e((4, 1)), e((4, 256), F), e((4, 2)), blocks(f8, e), blocks(f8, e, 48), 4, 32, 256)),
    "pair_into_few_rows": (ValueError, "codes / scales smaller",
        lambda f8, e: f8.gate_up(e((3, 32), F), e((4, 1)), e((4, 256), F), e((4, 2)), blocks(f8, e), blocks(f8, e), 4, 32, 256)),
    "pair_into_few_scales": (ValueError, "codes / scales smaller",
        lambda f8, e: f8.gate_up(e((4, 32), F), e((3, 1)), e((4, 256), F), e((4, 2)), blocks(f8, e), blocks(f8, e), 4, 32, 256)),
    "pair_of_odd_n": (HxError, "N must be",
        lambda f8, e: f8.gate_up(e((4, 24), F), e((4, 1)), e((4, 256), F), e((4, 2)), blocks(f8, e, 24), blocks(f8, e, 24), 4, 24, 256)),
    "pair_of_no_limit": (HxError, "limit",
        lambda f8, e: f8.gate_up(e((4, 32), F), e((4, 1)), e((4, 256), F), e((4, 2)), blocks(f8, e), blocks(f8, e), 4, 32, 256, limit=0.0)),
    "quantize_of_bf16": (ValueError, "float16 or float32", lambda f8, e: f8.quantize(e((4, 256), torch.bfloat16), e((4, 256), F), e((4, 2)), 4, 256)),
    "quantize_of_short_rows": (ValueError, "smaller than", lambda f8, e: f8.quantize(e((4, 128)), e((4, 256), F), e((4, 2)), 4, 256)),
    "quantize_of_columns": (ValueError, "consecutive", lambda f8, e: f8.quantize(e((256, 4)).t(), e((4, 256), F), e((4, 2)), 4, 256)),
    "quantize_of_one_row_again_and_again": (ValueError, "consecutive",
        lambda f8, e: f8.quantize(e((1, 256)).expand(4, 256), e((4, 256), F), e((4, 2)), 4, 256)),
    "quantize_of_rows_off_alignment": (HxError, "ld must be", lambda f8, e: f8.quantize(e((4, 260))[:, :256], e((4, 256), F), e((4, 2)), 4, 256)),
    "quantize_of_a_first_column_off_alignment": (HxError, "16-byte",
        lambda f8, e: f8.quantize(e((4, 264))[:, 2:258], e((4, 256), F), e((4, 2)), 4, 256)),
    "quantize_of_short_k": (HxError, "multiple of 16", lambda f8, e: f8.quantize(e((4, 40)), e((4, 40), F), e((4, 1)), 4, 40)),
    # messages name the argument
    "gemm_of_codes_in_fp32": (ValueError, "^x has dtype", lambda f8, e: f8.gemm(e((4, 32)), e((4, 256)), e((4, 2)), blocks(f8, e), 4, 32, 256, True)),
    "gemm_of_fp16_scales": (ValueError, "^x_scales has dtype",
        lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((4, 2), H), blocks(f8, e), 4, 32, 256, True)),
    "gemm_of_few_scales_of_x": (ValueError, ": x, x_scales$",
        lambda f8, e: f8.gemm(e((4, 32)), e((4, 256), F), e((3, 2)), blocks(f8, e), 4, 32, 256, True)),
    "pair_of_codes_in_fp32": (ValueError, "^x has dtype",
        lambda f8, e: f8.gate_up(e((4, 32), F), e((4, 1)), e((4, 256)), e((4, 2)), blocks(f8, e), blocks(f8, e), 4, 32, 256)),
    "pair_into_fp16_scales": (ValueError, "^scales has dtype",
        lambda f8, e: f8.gate_up(e((4, 32), F), e((4, 1), H), e((4, 256), F), e((4, 2)), blocks(f8, e), blocks(f8, e), 4, 32, 256)),
    "norm_with_a_short_weight": (ValueError, "K values", lambda f8, e: f8.rms_norm(e((4, 256)), e((255,)), 4, 256, 1e-5, y=e((4, 256), H))),
    "norm_without_out": (ValueError, "together",
        lambda f8, e: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, residual=e((4, 256)), y=e((4, 256), H))),
    "norm_with_out_of_another_type": (ValueError, "out",
        lambda f8, e: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, residual=e((4, 256)), out=e((4, 256), H), y=e((4, 256), H))),
    "norm_without_scales": (ValueError, "together",
        lambda f8, e: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, y=e((4, 256), H), q=e((4, 256), F))),
    "norm_into_fp32": (ValueError, "y", lambda f8, e: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5, y=e((4, 256)))),
    "norm_into_nothing": (HxError, "neither", lambda f8, e: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, 1e-5)),
    "norm_of_negative_eps": (HxError, "eps", lambda f8, e: f8.rms_norm(e((4, 256)), e((256,)), 4, 256, -1.0, y=e((4, 256), H))),
}


@pytest.mark.parametrize("case", REFUSALS)
def test_refusal(f8, case):
    kind, text, call = REFUSALS[case]
    with pytest.raises(kind, match=text):
        call(f8, lambda shape, dt=torch.float32: torch.zeros(shape, dtype=dt, device="cuda"))
    torch.cuda.synchronize()
