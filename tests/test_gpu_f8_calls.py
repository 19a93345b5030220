"""Calls of the 8-bit operators at the edges of what they take: rows past one launch, NaNs around and inside fp16 outputs' inputs, refusals."""
import numpy as np
import pytest

from test_gpu_f8 import check_blocks, f8, gated, host, inputs, weights  # noqa: F401

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
