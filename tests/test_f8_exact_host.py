"""Argument checks of the linear with exact products (nothing is launched)."""
import ctypes as C

import pytest
import torch

from helios_glm53flash_amd import _lib, f8

from test_f8_host import EXTENTS, FAR, WEIGHTS, blocks, err


@pytest.mark.parametrize("bad,text", EXTENTS + WEIGHTS + [
    (dict(y=None), "null"), (dict(x=None), "null"), (dict(xs=None), "null"), (dict(x=2 * FAR + 8), "16-byte"), (dict(xs=2), "aligned"),
    (dict(y=FAR + 1), "aligned"), (dict(y=2 * FAR), "overlap"), (dict(y=3 * FAR + 28), "overlap"), (dict(y=5 * FAR + 4), "overlap")])
def test_refusals(bad, text):
    a = dict(y=FAR, x=2 * FAR, xs=3 * FAR, M=4, N=100, K=256, w=None)
    a.update(bad)
    r = _lib.lib.hx_f8_gemm_exact(a["y"], a["x"], a["xs"], blocks(**(a["w"] or {})), a["M"], a["N"], a["K"], 0, None, None, 0)
    assert r == _lib.HX_ERR_INVALID and text in err() and err().startswith("hx_f8_gemm_exact: "), err()


def test_workspace_and_no_rows():
    w = C.byref(_lib.F8BlocksC(4 * FAR, 5 * FAR))
    assert _lib.lib.hx_f8_gemm_exact(FAR, 2 * FAR, 3 * FAR, w, 4, 100, 256, 0, None, 8, 0) == _lib.HX_ERR_WORKSPACE
    assert err() == "hx_f8_gemm_exact: workspace must be 16-byte aligned"
    assert _lib.lib.hx_f8_gemm_exact(None, None, None, w, 0, 100, 256, 0, None, None, 0) == 0


def test_python_checks():
    codes, scales = torch.zeros((4, 32), dtype=torch.float8_e4m3fn), torch.ones((1, 1))
    with pytest.raises(ValueError, match="32 bits"):
        f8.gemm(scales, codes, scales, None, 1 << 31, 4, 32, exact=True)


@pytest.mark.parametrize("M,N,K", [(1, 2048, 4096), (8, 16, 16), (12, 144, 400), (33, 1040, 2704)])
def test_gated_pair_without_its_workspace(M, N, K):
    """Sizes whose blocks of outputs meet in memory: the size is not 0, and a call with less, none or a misaligned one is refused."""
    need = _lib.lib.hx_f8_gate_up_workspace_size(M, N, K)
    assert need > 64 * 1024
    w = C.byref(_lib.F8BlocksC(400 * FAR, 500 * FAR))
    for ws, size in ((None, need), (700 * FAR + 8, need), (700 * FAR, need - 1), (700 * FAR, 0)):
        r = _lib.lib.hx_f8_gate_up(FAR, 100 * FAR, 200 * FAR, 300 * FAR, w, w, M, N, K, 10.0, None, ws, size)
        assert r == _lib.HX_ERR_WORKSPACE and "hx_f8_gate_up_workspace_size" in err(), (ws, size, err())
