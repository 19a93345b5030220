"""Host side of the 8-bit block-scaled linear, its gated pair, the norm and the quantization: argument checks (nothing is launched)."""
import ctypes as C

import pytest
import torch

from helios_glm53flash_amd import _lib, f8

LIB = _lib.lib
FAR = 1 << 30  # addresses that are never touched, far apart


def err():
    return LIB.hx_last_error().decode()


def refused(r, text):
    assert r == _lib.HX_ERR_INVALID and text in err(), (r, err())


def quantize(**kw):
    a = dict(x=FAR, q=2 * FAR, scales=3 * FAR, M=4, K=256, ld=256, dtype=0)
    a.update(kw)
    return LIB.hx_f8_quantize(*a.values(), None)


EXTENTS = [(dict(M=-1), "negative"), (dict(K=0), "multiple of 16"), (dict(K=-16), "multiple of 16"), (dict(K=24), "multiple of 16"),
           (dict(K=(1 << 22) + 16), "2^22")]


@pytest.mark.parametrize("bad,text", EXTENTS + [
    (dict(dtype=2), "dtype"), (dict(ld=248), "ld"), (dict(ld=257), "ld"), (dict(ld=-256), "ld"), (dict(ld=1 << 40), "ld"), (dict(x=None), "null"),
    (dict(q=None), "null"), (dict(scales=None), "null"), (dict(x=FAR + 8), "16-byte"), (dict(q=FAR + 8), "16-byte"),
    (dict(scales=FAR + 2), "4-byte"), (dict(q=FAR), "overlap"), (dict(q=FAR + 2048 - 16), "overlap"), (dict(q=FAR - 1024 + 16), "overlap"),
    (dict(scales=FAR), "overlap"), (dict(scales=2 * FAR + 1020), "overlap"), (dict(q=FAR + 2048, dtype=1), "overlap"),
    (dict(q=FAR + 1024, M=2, ld=512), "overlap")])
def test_quantize_refusals(bad, text):
    refused(quantize(**bad), text)


def test_no_rows():
    assert quantize(M=0, x=None, q=None, scales=None) == 0
    assert norm(M=0, x=None, weight=None, residual=None, out=None, y=None, q=None, scales=None) == 0
    assert gemm(M=0, x=None, xs=None, y=None) == 0
    assert gate_up(M=0, x=None, xs=None, q=None, scales=None) == 0


def norm(**kw):
    a = dict(x=FAR, ld=256, xd=0, residual=2 * FAR, out=3 * FAR, rd=0, weight=4 * FAR, wd=0, y=5 * FAR, q=6 * FAR, scales=7 * FAR, M=4,
             K=256, eps=1e-5)
    a.update(kw)
    return LIB.hx_f8_rms_norm(*a.values(), None)


@pytest.mark.parametrize("bad,text", EXTENTS + [
    (dict(xd=2), "dtype"), (dict(rd=-1), "dtype"), (dict(wd=7), "dtype"), (dict(ld=128), "ld"), (dict(ld=260), "ld"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=None), "null"), (dict(weight=None), "null"),
    (dict(residual=None), "together"), (dict(out=None), "together"), (dict(q=None), "together"), (dict(scales=None), "together"),
    (dict(y=None, q=None, scales=None), "neither"), (dict(x=FAR + 8), "16-byte"), (dict(y=FAR + 2), "16-byte"),
    (dict(weight=4 * FAR + 4), "16-byte"), (dict(scales=1), "4-byte"), (dict(out=FAR), "an output overlaps an input"),
    (dict(out=2 * FAR + 16), "an output overlaps an input"), (dict(y=2 * FAR), "an output overlaps an input"),
    (dict(q=4 * FAR + 496), "an output overlaps an input"), (dict(y=3 * FAR), "outputs overlap"), (dict(scales=6 * FAR), "outputs overlap")])
def test_norm_refusals(bad, text):
    refused(norm(**bad), text)


def blocks(codes=4 * FAR, scales=5 * FAR, null=False):
    return None if null else C.byref(_lib.F8BlocksC(codes, scales))


def gemm(w=None, **kw):
    a = dict(y=FAR, x=2 * FAR, xs=3 * FAR, M=4, N=100, K=256, fp32=1, ws=None)
    a.update(kw)
    return LIB.hx_f8_gemm(a["y"], a["x"], a["xs"], blocks(**(w or {})), a["M"], a["N"], a["K"], a["fp32"], None, a["ws"], 0)


WEIGHTS = [(dict(w=dict(null=True)), "null"), (dict(w=dict(codes=None)), "null"), (dict(w=dict(scales=None)), "null"),
           (dict(w=dict(codes=8)), "16-byte"), (dict(w=dict(scales=2)), "4-byte"), (dict(N=0), "N must"), (dict(N=-16), "N must"),
           (dict(N=(1 << 28) + 16), "N must")]


@pytest.mark.parametrize("bad,text", EXTENTS + WEIGHTS + [
    (dict(y=None), "null"), (dict(x=None), "null"), (dict(xs=None), "null"), (dict(x=2 * FAR + 8), "16-byte"), (dict(xs=2), "aligned"),
    (dict(y=FAR + 2), "aligned"), (dict(y=FAR + 1, fp32=0), "aligned"), (dict(y=2 * FAR), "overlap"), (dict(y=2 * FAR - 1596), "overlap"),
    (dict(y=2 * FAR + 1020), "overlap"), (dict(y=3 * FAR + 28), "overlap"),
    (dict(y=4 * FAR + 25584), "overlap"), (dict(y=5 * FAR + 4), "overlap")])
def test_gemm_refusals(bad, text):
    refused(gemm(**bad), text)


def test_gemm_workspace_alignment():
    assert gemm(ws=8) == _lib.HX_ERR_WORKSPACE and "16-byte" in err()


def gate_up(w=None, w2=None, **kw):
    a = dict(q=FAR, scales=6 * FAR, x=2 * FAR, xs=3 * FAR, M=4, N=256, K=256, limit=10.0, ws=7 * FAR, bytes=1 << 30)
    a.update(kw)
    return LIB.hx_f8_gate_up(a["q"], a["scales"], a["x"], a["xs"], blocks(**(w or {})), blocks(**(w2 or {})), a["M"], a["N"], a["K"],
                             a["limit"], None, a["ws"], a["bytes"])


@pytest.mark.parametrize("bad,text", EXTENTS + WEIGHTS + [
    (dict(w2=dict(null=True)), "null"), (dict(w2=dict(codes=8)), "16-byte"), (dict(N=200), "multiple of 16"), (dict(limit=0.0), "limit"),
    (dict(limit=float("nan")), "limit"), (dict(limit=-1.0), "limit"), (dict(q=None), "null"), (dict(scales=None), "null"),
    (dict(x=None), "null"), (dict(xs=None), "null"), (dict(q=FAR + 8), "16-byte"), (dict(scales=6 * FAR + 1), "4-byte"),
    (dict(q=2 * FAR - 16), "an output overlaps an input"), (dict(scales=3 * FAR + 28), "an output overlaps an input"),
    (dict(scales=FAR + 1020), "outputs overlap"), (dict(q=4 * FAR + 65520), "an output overlaps an input"),
    (dict(scales=5 * FAR + 12), "an output overlaps an input"), (dict(w2=dict(codes=FAR - 65520)), "an output overlaps an input")])
def test_gate_up_refusals(bad, text):
    refused(gate_up(**bad), text)


def test_workspace_sizes():
    for size in (LIB.hx_f8_gemm_workspace_size, LIB.hx_f8_gate_up_workspace_size):
        for bad in ((0, 256, 256), (-1, 256, 256), (4, 0, 256), (4, 256, 0), (4, 256, 8), (4, (1 << 28) + 16, 256), (4, 256, (1 << 22) + 16)):
            assert size(*bad) == 0
    need = LIB.hx_f8_gate_up_workspace_size(1, 2048, 4096)
    if need:
        for bad in (dict(ws=None), dict(ws=7 * FAR + 8), dict(bytes=need - 1)):
            assert gate_up(M=1, N=2048, K=4096, w=dict(scales=50 * FAR), w2=dict(scales=50 * FAR), **bad) == _lib.HX_ERR_WORKSPACE


def test_python_checks():
    codes, scales = torch.zeros((4, 32), dtype=torch.float8_e4m3fn), torch.ones((1, 1))
    with pytest.raises(ValueError, match="device tensor"):
        f8.F8Blocks(codes, scales)
    with pytest.raises(TypeError):
        f8.F8Blocks(None, scales)
    x = torch.zeros((2, 32), dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensor"):
        f8.quantize(x, codes, scales, 2, 32)
    with pytest.raises(ValueError, match="device tensor"):
        f8.rms_norm(x, x[0], 2, 32, 1e-5, q=codes, scales=scales)
    with pytest.raises(ValueError, match="32 bits"):
        f8.quantize(x, codes, scales, -1, 32)
    with pytest.raises(ValueError, match="32 bits"):
        f8.gemm(x, codes, scales, None, 1 << 31, 4, 32)
