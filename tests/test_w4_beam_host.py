"""Host side of the 4-bit linear and of beam search: the words' layout, argument checks (nothing is launched)."""
import ctypes as C

import numpy as np
import pytest
import torch

from helios_glm53flash_amd import _lib, beam, w4

LIB = _lib.lib


def err():
    return LIB.hx_last_error().decode()


@pytest.mark.parametrize("N,K", [(1, 32), (3, 128), (5, 160), (2, 4096), (7, 992)])
def test_words_follow_the_documented_layout(N, K):
    q = np.random.default_rng(K).integers(0, 16, (N, K), dtype=np.uint8)
    words = w4.pack(torch.from_numpy(q))
    assert words.dtype == torch.int32 and words.shape == (N, (K + 127) // 128 * 16)
    u = words.numpy().view(np.uint32)
    want = np.zeros_like(u)
    for k in range(K):
        block, j, g, o = k // 128, k % 128 // 32, k % 32 // 8, k % 8
        want[:, 16 * block + 4 * g + j] |= q[:, k].astype(np.uint32) << np.uint32(4 * (o // 2 + 4 * (o % 2)))
    assert np.array_equal(u, want)
    assert np.array_equal(w4.unpack(words, K).numpy(), q)


def test_pack_refusals():
    with pytest.raises(ValueError):
        w4.pack(torch.zeros((2, 100), dtype=torch.uint8))
    with pytest.raises(ValueError):
        w4.pack(torch.zeros((2, 0), dtype=torch.uint8))
    with pytest.raises(ValueError):
        w4.pack(torch.full((2, 32), 16, dtype=torch.uint8))
    with pytest.raises(ValueError):
        w4.pack(torch.zeros((2, 32)))
    with pytest.raises(ValueError):
        w4.unpack(torch.zeros((2, 15), dtype=torch.int32), 128)
    assert w4.pack(torch.zeros((0, 64), dtype=torch.uint8)).shape == (0, 16)


def gemm(y=16, x=16, words=16, scales=16, zeros=None, group=64, M=1, N=16, K=128, null=False, ws=None):
    w = _lib.W4WordsC(words, scales, zeros, group)
    return LIB.hx_w4_gemm(y, x, None if null else C.byref(w), M, N, K, 1, None, ws, 1 << 30)


@pytest.mark.parametrize("bad,text", [
    (dict(null=True), "null"), (dict(words=None), "null"), (dict(scales=None), "null"), (dict(y=None), "null"),
    (dict(x=None), "null"), (dict(K=100), "multiple of 32"), (dict(K=0), "positive"), (dict(K=-128), "positive"),
    (dict(N=0), "positive"), (dict(M=-1), "negative"), (dict(group=16), "power of two"), (dict(group=96), "power of two"),
    (dict(group=0), "power of two"), (dict(group=-64), "power of two"), (dict(words=24), "16-byte"), (dict(x=8), "16-byte"),
    (dict(y=18), "aligned"), (dict(scales=17), "aligned"), (dict(K=(1 << 22) + 32), "2^22")])
def test_gemm_refusals(bad, text):
    assert gemm(**bad) == _lib.HX_ERR_INVALID and text in err()


def test_gemm_of_no_rows():
    assert gemm(M=0, x=None, y=None) == 0


@pytest.mark.parametrize("bad,text", [(dict(n=-1), "negative"), (dict(out=None), "null"), (dict(tokens=None), "null"),
                                      (dict(out=8), "16-byte"), (dict(tokens=4), "8-byte"), (dict(K=48), "multiple of 32")])
def test_embed_refusals(bad, text):
    a = dict(tokens=16, out=16, n=1, N=16, K=128)
    a.update(bad)
    w = _lib.W4WordsC(16, 16, None, 64)
    r = LIB.hx_w4_embed(C.byref(w), a["tokens"], a["out"], a["n"], a["N"], a["K"], 1.0, 1, None)
    assert r == _lib.HX_ERR_INVALID and text in err()
    assert LIB.hx_w4_embed(C.byref(w), None, None, 0, 16, 128, 1.0, 1, None) == 0


def select(**kw):
    a = dict(logits=16, cum=16, done=None, scores=16, parents=16, tokens=16, batch=1, beams=4, vocab=100, n=8, ld=100, eos=0,
             dtype=1, stream=None, ws=16, bytes=1 << 30)
    a.update(kw)
    return LIB.hx_beam_select(*a.values())


@pytest.mark.parametrize("bad,text", [
    (dict(batch=-1), "batch"), (dict(batch=4097), "batch"), (dict(beams=0), "positive"), (dict(beams=1025), "1024"),
    (dict(vocab=0), "positive"), (dict(n=0), "n in"), (dict(n=129), "n in"), (dict(ld=99), "ld"), (dict(dtype=2), "dtype"),
    (dict(done=16, eos=100), "eos"), (dict(done=16, eos=-1), "eos"), (dict(logits=None), "null"), (dict(cum=None), "null"),
    (dict(scores=None), "null"), (dict(parents=None), "null"), (dict(tokens=None), "null"), (dict(logits=18), "aligned"),
    (dict(parents=20), "aligned"), (dict(cum=18), "aligned")])
def test_select_refusals(bad, text):
    assert select(**bad) == _lib.HX_ERR_INVALID and text in err()


def test_select_workspace():
    assert select(ws=None) == _lib.HX_ERR_WORKSPACE and select(ws=24) == _lib.HX_ERR_WORKSPACE
    need = LIB.hx_beam_select_workspace_size(3, 4, 5000, 8)
    assert need > 65536
    assert select(batch=3, vocab=5000, ld=5000, bytes=need - 1) == _lib.HX_ERR_WORKSPACE
    assert select(batch=0, logits=None, cum=None, scores=None, parents=None, tokens=None, ws=None, bytes=0) == 0
    assert LIB.hx_beam_select_workspace_size(0, 4, 5000, 8) == 0


def reorder(src=1 << 20, dst=1 << 30, parents=16, batch=2, beams=3, out_beams=3, outer=1, inner=1, bytes=64,
            ss=(0, 64, 0), ds=(0, 64, 0)):
    t = C.c_int64 * 3
    return LIB.hx_beam_reorder(src, parents, dst, batch, beams, out_beams, outer, inner, bytes, t(*ss), t(*ds), None)


@pytest.mark.parametrize("bad,text", [
    (dict(batch=-1), "extent"), (dict(beams=0), "beams"), (dict(out_beams=-1), "extent"), (dict(bytes=-1), "extent"),
    (dict(src=None), "null"), (dict(dst=None), "null"), (dict(parents=None), "null"), (dict(parents=12), "aligned"),
    (dict(dst=1 << 20), "overlap"), (dict(dst=(1 << 20) + 6 * 64 - 1), "overlap"), (dict(dst=(1 << 20) - 6 * 64 + 1), "overlap"),
    (dict(ds=(0, 63, 0)), "overlap"), (dict(ds=(0, 0, 0)), "overlap"), (dict(ss=(0, -64, 0)), "negative"),
    (dict(ds=(0, -64, 0)), "negative"), (dict(outer=2, ds=(100, 64, 0)), "overlap"),
    (dict(inner=4, bytes=16, ss=(0, 64, 16), ds=(0, 60, 16)), "overlap"), (dict(ss=(0, 1 << 62, 0)), "negative"),
    (dict(outer=1 << 60, ss=(0, 64, 0), ds=(1, 64, 0)), "too large")])
def test_reorder_refusals(bad, text):
    assert reorder(**bad) == _lib.HX_ERR_INVALID and text in err()


@pytest.mark.parametrize("none", [dict(batch=0), dict(out_beams=0), dict(outer=0), dict(inner=0), dict(bytes=0)])
def test_reorder_of_nothing(none):
    assert reorder(src=None, dst=None, parents=None, **none) == 0


@pytest.mark.parametrize("shape,dim,view,want", [
    ((12, 7), 0, None, ((1, 0, 0), (1, 0, 0), 28)),
    ((3, 12, 5, 16), 1, None, ((3, 3840, 3840), (1, 0, 0), 320)),
    ((3, 12, 5, 16), 1, 4, ((3, 3840, 3840), (1, 0, 0), 256)),
    ((2, 3, 12, 4, 8, 6), 2, 5, ((6, 9216, 9216), (4, 192, 192), 120)),
    ((12,), 0, None, ((1, 0, 0), (1, 0, 0), 4))])
def test_reorder_merges_dimensions(shape, dim, view, want):
    t = torch.zeros(shape)
    if view is not None:
        t = t.narrow(-2, 0, view)
    dims = [(n, s * 4, s * 4) for n, s in zip(t.shape, t.stride())]
    inner, run = beam._merge(dims[dim + 1:], 4)
    outer, _ = beam._merge(dims[:dim], None)
    assert (outer, inner, run) == want


def test_reorder_refuses_irreducible_strides():
    t = torch.zeros((6, 4, 5, 8))[:, :3, :3, :6]
    dims = [(n, s * 4, s * 4) for n, s in zip(t.shape, t.stride())]
    with pytest.raises(ValueError):
        beam._merge(dims[1:], 4)


def test_gemm_workspace():
    size = LIB.hx_w4_gemm_workspace_size
    assert gemm(ws=24) == _lib.HX_ERR_WORKSPACE and "16-byte" in err()
    assert size(1, 4096, 8192) == 0 and size(0, 4096, 8192) == 0  # single tokens need none
    assert size(64, 4096, 8192) > 65536
    for M in (9, 16, 17, 32, 33, 64, 65, 128, 200, 512, 2000):
        for N in (1, 64, 2048, 4096, 12288, 151552):
            for K in (32, 2048, 4096, 16384, 1 << 22):
                assert size(M, N, K) <= 9 << 20, (M, N, K)


def test_extents_beyond_a_call():
    assert gemm(N=(1 << 28) + 1) == _lib.HX_ERR_INVALID and "2^28" in err()
    assert select(vocab=(1 << 30) + 1, ld=1 << 31) == _lib.HX_ERR_INVALID and "2^30" in err()
    assert LIB.hx_w4_gemm_workspace_size(64, (1 << 28) + 1, 128) == 0
    assert LIB.hx_w4_gemm_workspace_size((1 << 31) - 1, 64, 128) == 0
    assert LIB.hx_w4_gemm_workspace_size(64, 4096, (1 << 31) - 1) == 0
    assert LIB.hx_beam_select_workspace_size(1, 1, (1 << 31) - 1, 8) == 0


@pytest.mark.parametrize("kw", [dict(scores=16), dict(scores=28, n=4), dict(scores=4, n=4, beams=4), dict(scores=16, n=3, beams=4)])
def test_select_refuses_overlapping_scores(kw):
    assert select(**{"cum": 16, "n": 8, **kw}) == _lib.HX_ERR_INVALID and "overlap" in err()


def test_gemm_workspace_bound():
    """The counters and 256 workgroups' 64 x 64 fp32 sums: never more, and reached."""
    size, most = LIB.hx_w4_gemm_workspace_size, 65536 + 256 * 64 * 64 * 4
    assert size(33, 2048, 65536) == most
    for M in (9, 16, 17, 32, 33, 48, 64, 65, 128, 129, 256, 512, 600):
        for N in [64 * i + j for i in range(1, 70, 3) for j in (0, 1)] + [8192, 12288, 16384, 24576, 151552]:
            for K in (2048, 4096, 16384, 65536, 1 << 22):
                assert size(M, N, K) <= most, (M, N, K)
