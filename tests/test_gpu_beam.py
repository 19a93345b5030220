"""Beam search's selection and reordering through the C ABI against the definition in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def beam():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from helios_glm53flash_amd import beam
    return beam


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def reference(logits, cum, done, batch, beams, V, n, eos):
    """(scores float64, parents, tokens) [batch][n] by the definition."""
    out = np.full((batch, n), -np.inf), np.full((batch, n), -1, np.int64), np.full((batch, n), -1, np.int64)
    for b in range(batch):
        cand = []
        for w in range(beams):
            r = b * beams + w
            c = float(cum[r])
            if not np.isfinite(c):
                continue
            if done is not None and done[r]:
                cand.append((-c, w, eos))
                continue
            x = logits[r, :V].astype(np.float64)
            top = x.max()
            if not np.isfinite(top):
                continue
            # relative to the maximum: top + log(sum) would lose the logarithm beside a large top
            lsum = np.log(np.exp(x - top).sum())
            at = np.argsort(-x, kind="stable")[:n]
            cand += [(-(c + ((x[t] - top) - lsum)), w, int(t)) for t in at if x[t] > -np.inf]
        for i, (s, w, t) in enumerate(sorted(cand)[:n]):
            out[0][b, i], out[1][b, i], out[2][b, i] = -s, w, t
    return out


# Error of a score: the log-sum-exp holds exponentials of fp32 arguments.  Each term's argument x - max (of size t) is off by
# at most t 2^-23 and its exponential by 2^-22 relative, and the terms' weighted mean of t is at most ln(vocab) + 1 < 13:
# 13 x 2^-23 + 2^-22 = 1.8e-6; 64 fp32 additions per thread at most: 64 x 2^-24 = 3.8e-6.  Then the fp32 rounding of the score.
LSE_TOL = 6e-6


def check(beam, logits, cum, done, batch, beams, V, n, eos=0, ld=None):
    import torch
    lt = logits if isinstance(logits, torch.Tensor) else dev(logits)
    ln = lt.cpu().numpy()
    s = torch.full((batch + 2, n), 9.0, device="cuda")
    p = torch.full((batch + 2, n), 9, dtype=torch.int64, device="cuda")
    t = torch.full((batch + 2, n), 9, dtype=torch.int64, device="cuda")
    beam.select(lt, dev(cum), dev(done) if done is not None else None, s[1:-1], p[1:-1], t[1:-1], batch, beams, V, n, eos)
    torch.cuda.synchronize()
    for o in (s, p, t):
        assert bool((o[0] == 9).all()) and bool((o[-1] == 9).all())
    s, p, t = (o[1:-1].cpu().numpy() for o in (s, p, t))
    rs, rp, rt = reference(ln, cum, done, batch, beams, V, n, eos)
    none = rs == -np.inf
    assert np.array_equal(s == -np.inf, none)
    assert (p[none] == -1).all() and (t[none] == -1).all()
    tol = np.where(none, 0.0, LSE_TOL + 2.0 ** -24 * np.abs(np.where(none, 0.0, rs)))
    with np.errstate(invalid="ignore"):
        assert (np.abs(np.where(none, 0.0, s - rs)) <= tol).all()
    # ranks of different beams closer than the error of their scores may swap; all others are fixed
    for b in range(batch):
        for i in range(n):
            if none[b, i] or (p[b, i], t[b, i]) == (rp[b, i], rt[b, i]):
                continue
            near = [j for j in range(n) if j != i and abs(rs[b, j] - rs[b, i]) <= 2 * LSE_TOL and rp[b, j] != rp[b, i]]
            last_near = i >= n - 1 or any(j == n - 1 for j in near)
            assert near or last_near, (b, i, p[b], rp[b], t[b], rt[b])
            assert any((p[b, i], t[b, i]) == (rp[b, j], rt[b, j]) for j in near), (b, i)
        pairs = [(int(a), int(c)) for a, c in zip(p[b], t[b]) if a >= 0]
        assert len(set(pairs)) == len(pairs)
    return s, p, t


def data(seed, rows, V, dtype, scale=3.0):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((rows, V)) * scale).astype(np.float32)
    x[r.random((rows, V)) < 0.01] = -np.inf
    return x.astype(dtype), (-r.uniform(0, 6, rows)).astype(np.float32)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch,beams,V,n", [
    (1, 1, 1, 1), (1, 1, 1, 5), (1, 4, 2, 8), (1, 4, 151552, 8), (3, 5, 1000, 10), (2, 8, 50257, 16), (7, 3, 4097, 6),
    (40, 2, 333, 4), (1, 64, 2500, 128), (2, 16, 20001, 32), (5, 1, 70000, 1), (2, 100, 777, 128), (1, 2, 65, 128),
    (300, 1, 130, 2), (1, 1024, 40, 128), (1, 1, 300000, 128)])
def test_select(beam, dtype, batch, beams, V, n):
    x, cum = data(batch * 7 + V, batch * beams, V, dtype)
    check(beam, x, cum, None, batch, beams, V, n)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_select_done_and_dead_beams(beam, dtype):
    batch, beams, V, n = 6, 6, 3000, 12
    x, cum = data(5, batch * beams, V, dtype)
    done = (np.random.default_rng(1).random(batch * beams) < 0.4).astype(np.uint8)
    done[:6] = 1                      # every beam of the first sequence is finished
    done[6:12] = 0
    cum[6:12] = -np.inf               # and every beam of the second is dead
    done[12:18], cum[13:18] = 0, -np.inf  # the first step of the third: one live beam
    cum[18], cum[19], cum[20] = np.nan, np.inf, -np.inf
    done[24] = 255
    s, p, t = check(beam, x, cum, done, batch, beams, V, n, eos=7)
    assert (p[1] == -1).all() and (p[2] == 0).all() and (t[0][:6] == 7).all() and (t[0][6:] == -1).all()
    check(beam, x, cum, done, batch, beams, V, n, eos=V - 1)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_select_rows_without_candidates(beam, dtype):
    """Rows of -inf, with a NaN, with +inf, of the type's lowest value; a single finite logit."""
    V, n = 5000, 6
    x, cum = data(9, 8, V, dtype)
    x[0] = -np.inf
    x[1, 4999] = np.nan
    x[2, 0] = np.inf
    x[3] = np.finfo(dtype).min
    x[4] = -np.inf
    x[4, 4321] = -3.0
    x[5] = np.finfo(dtype).max
    x[6, 100:] = -np.inf
    s, p, t = check(beam, x, cum, None, 8, 1, V, n)
    for r in (0, 1, 2):
        assert (p[r] == -1).all()
    assert np.array_equal(t[3], np.arange(n)) and np.array_equal(t[5], np.arange(n))
    assert t[4][0] == 4321 and (t[4][1:] == -1).all()
    check(beam, x, cum, None, 1, 8, V, 40)
    check(beam, x, cum, None, 2, 4, V, 100)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("V,n", [(40000, 16), (151552, 128), (600, 100)])
def test_select_equal_logits_go_to_the_lowest_token(beam, dtype, V, n):
    """Rows of few distinct values, constant rows, and ties over the whole row; equal beams go to the lowest beam."""
    r = np.random.default_rng(V)
    x = np.zeros((6, V), dtype)
    x[1] = r.integers(0, 3, V)
    x[2] = np.where(np.arange(V) >= V - 5, 2.0, 1.0)
    x[3] = (np.arange(V) // 100).astype(dtype)[::-1]
    x[4] = x[1]
    x[5] = -0.0
    x[5, ::2] = 0.0
    cum = np.zeros(6, np.float32)
    cum[4] = cum[1]
    s, p, t = check(beam, x, cum, None, 6, 1, V, n)
    for i in range(6):
        at = np.argsort(-x[i].astype(np.float64), kind="stable")[:n]
        assert np.array_equal(t[i], at)
    two = np.concatenate([x[1:2], x[1:2]])
    s, p, t = check(beam, two, np.full(2, -1.0, np.float32), None, 1, 2, V, n)
    at = np.argsort(-x[1].astype(np.float64), kind="stable")
    top = at[x[1][at] == 2][:n]  # the tied tokens of the first beam, then those of the second
    k = min(n, len(top))
    assert np.array_equal(t[0][:k], top[:k]) and (p[0][:k] == 0).all()


def shaped_rows(r, rows, V, dtype):
    """Rows that a bound found on the way meets in every manner: ascending and descending, equal in all or most places, steps
    of hundreds of equal logits, the largest at the very end or start, hardly any finite, of the type's lowest value."""
    x = (r.standard_normal((rows, V)) * 3).astype(np.float32)
    ramp = np.arange(V) * np.float32(60.0 / V)
    x[1::11] = ramp
    x[2::11] = -ramp
    x[3::11] = np.floor(ramp)
    x[4::11] = -np.floor(ramp)
    x[5::11] = -1.5
    x[6::11] = r.integers(0, 3, x[6::11].shape)
    x[7::11, V - 7:] += 30
    x[8::11] = np.where(r.random(x[8::11].shape) < 0.0005, x[8::11], -np.inf)
    x[9::11] = np.where(r.random(x[9::11].shape) < 0.5, x[9::11], -np.inf)
    x = x.astype(dtype)
    x[10::11] = np.finfo(dtype).min
    x[10::22, V // 2:] = 1.0
    x[1, -1], x[12, V // 2], x[23, 0] = np.nan, np.inf, -np.inf
    return x


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch,beams,V,n", [(600, 1, 20001, 1), (600, 1, 20001, 128), (130, 4, 33000, 33), (260, 2, 8193, 8),
                                             (1, 520, 12289, 128), (520, 1, 36864, 20)])
def test_select_many_rows(beam, dtype, batch, beams, V, n):
    """More rows than workgroups fit the chip, so that a workgroup walks over several pieces of its row."""
    r = np.random.default_rng(V + n)
    x = shaped_rows(r, batch * beams, V, dtype)
    cum = (-r.uniform(0, 6, batch * beams)).astype(np.float32)
    check(beam, x, cum, None, batch, beams, V, n)


# The bound on a log-sum-exp does not grow with the logits: exponentials are relative to the largest, and each change of what
# they are relative to is a factor of 2^(a difference of two fp32 values), 2^-23 off.  A thread here meets up to 3 such changes.
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("offset", [0.0, 20.0, -100.0, 300.0, 1000.0, -3000.0, 30000.0, -60000.0, 60000.0, 1e6])
def test_select_of_logits_far_from_zero(beam, dtype, offset):
    """Rows about a common offset: normal ones, one logit above a constant row, two finite logits in different threads, waves or
    pieces, steps up and down; alone, and as beams whose best scores differ by 1e-4."""
    if dtype == np.float16 and abs(offset) > 60000:
        pytest.skip("beyond fp16")
    r = np.random.default_rng(int(abs(offset)) + 3)
    for batch, V in ((3, 151552), (65, 12289)):  # chunks of one piece, and workgroups that walk over four
        rows = 8 * batch
        x = np.full((rows, V), offset, np.float32)
        x[0::8] += r.standard_normal(x[0::8].shape).astype(np.float32) * 3
        step = max(3.0, 1.001 * float(np.spacing(dtype(abs(offset)))))
        at = r.integers(0, V, rows)
        x[np.arange(rows), at] += step
        x[2::8] += np.arange(V) // (V // 5) * np.float32(step)
        x[3::8] -= np.arange(V) // (V // 5) * np.float32(step)
        x[4::8, 0] = offset + step
        for i, gap in ((5, 16), (6, 1024), (7, V - 1)):  # all of the row but two logits forbidden
            two = np.full_like(x[i::8], -np.inf)
            two[:, 0], two[:, gap] = offset, offset + step
            x[i::8] = two
        x = x.astype(dtype)
        x64 = x.astype(np.float64)
        top = x64.max(axis=1)
        best = -np.log(np.exp(x64 - top[:, None]).sum(axis=1))
        cum = np.zeros(rows, np.float32)
        check(beam, x, cum, None, rows, 1, V, 5)
        want = -20.0 + 1e-4 * r.permuted(np.tile(np.arange(8), (batch, 1)), axis=1).reshape(-1)
        check(beam, x, (want - best).astype(np.float32), None, batch, 8, V, 16)


def test_select_large_vocabulary(beam):
    """300 million tokens: places next to both ends and around multiples of the pieces that workgroups read."""
    import torch
    V, n = 300_000_001, 12
    x = torch.zeros((1, V), dtype=torch.float16, device="cuda")
    at = [0, 1, 4095, 4096, (1 << 28) - 1, 1 << 28, V - 1, V - 2, 299_999_232, 123_456_789, 4096 * 5000, 7]
    for i, a in enumerate(at):
        x[0, a] = 12.0 - i * 0.5
    s, p, t = (torch.empty((1, n), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64))
    beam.select(x, torch.zeros(1, device="cuda"), None, s, p, t, 1, 1, V, n)
    assert t[0].tolist() == at and bool((p == 0).all())
    v = 12.0 - 0.5 * np.arange(n)
    lse = np.log(np.exp(v).sum() + (V - n))
    # a thread adds some thousand exponentials of fp32: a relative error of 4096 x 2^-24 at most
    assert (np.abs(s[0].cpu().numpy() - (v - lse)) <= 2.5e-4).all()


def test_extents_beyond_32_bits_are_refused(beam):
    """They would reach the C entries modulo 2^32: an eos of 2^32 + 5 as 5, a vocabulary of 2^32 + 100 tokens as 100."""
    import torch
    V = 50
    cum, done = torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.uint8, device="cuda")
    out = [torch.full((1, 2), 9, dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64)]
    x = torch.randn((2, V), device="cuda")
    for eos in ((1 << 32) + 5, -(1 << 32), 1 << 31):
        with pytest.raises(ValueError, match="32 bits"):
            beam.select(x, cum, done, *out, 1, 2, V, 2, eos)
    big = torch.zeros((1, (1 << 32) + 100), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        beam.select(big, cum[:1], None, *out, 1, 1, big.shape[1], 2)
    rows = big.view(-1, 1)
    with pytest.raises(ValueError, match="32 bits"):
        beam.select(rows, cum, None, *out, rows.shape[0], 1, 1, 2)
    with pytest.raises(ValueError, match="32 bits"):
        beam.select(x, cum, None, *out, 1, 2, V, 1 << 32)
    assert all(bool((o == 9).all()) for o in out)
    parents = torch.zeros((1, 2), dtype=torch.int64, device="cuda")
    for extents in ((1 << 32, 1, 1), (1, 1 << 32, 1), (1, 1, 1 << 32)):
        with pytest.raises(ValueError, match="32 bits"):
            beam.reorder(x, parents, torch.zeros_like(x), *extents)


def test_select_scores_in_place_of_cum(beam):
    import torch
    batch, beams, V = 5, 6, 20000
    x = torch.randn((batch * beams, V), device="cuda") * 3
    cum = -torch.rand((batch, beams), device="cuda")
    want = [torch.empty((batch, beams), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64)]
    got = [torch.empty_like(o) for o in want]
    beam.select(x, cum, None, *want, batch, beams, V, beams)
    beam.select(x, cum, None, cum, *got[1:], batch, beams, V, beams)
    assert torch.equal(cum, want[0]) and all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


def test_select_padded_and_strided_rows(beam):
    """Rows at a stride beyond the vocabulary, starting at any element: what lies between them is never read into a result."""
    import torch
    V = 1237
    for dtype in (torch.float32, torch.float16):
        for off, pad in ((0, 3), (1, 2), (3, 64), (5, 1)):
            whole = torch.full((12, off + V + pad), float("nan"), dtype=dtype, device="cuda")
            whole[:, off:off + V] = torch.randn((12, V), device="cuda") * 3
            view = whole[:, off:off + V]
            check(beam, view, (-np.arange(12) * 0.37).astype(np.float32), None, 3, 4, V, 8)
            check(beam, view[::2], (-np.arange(6) * 0.37).astype(np.float32), None, 3, 2, V - 6, 8)


def test_select_large_rows_offsets(beam):
    """Rows whose offset passes 2^31 elements."""
    import torch
    rows, ld, V = 4, 800_000_000, 5000
    whole = torch.empty(3 * ld + V, dtype=torch.float16, device="cuda")
    view = whole.as_strided((rows, V), (ld, 1))
    view.copy_(torch.randn((rows, V), device="cuda") * 3)
    s, p, t = (torch.empty((1, 8), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64))
    cum = torch.tensor([-3.0, -2.0, -1.0, 0.0], device="cuda")
    beam.select(view, cum, None, s, p, t, 1, rows, V, 8)
    s2, p2, t2 = (torch.empty_like(o) for o in (s, p, t))
    beam.select(view.clone(), cum, None, s2, p2, t2, 1, rows, V, 8)
    assert torch.equal(s, s2) and torch.equal(p, p2) and torch.equal(t, t2)


def test_select_graph_and_streams(beam):
    """Captured calls replay on new logits; two streams at once have workspaces of their own."""
    import torch
    batch, beams, V, n = 4, 4, 30000, 8
    def outs():
        return [torch.empty((batch, n), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64)]
    x = torch.randn((batch * beams, V), device="cuda") * 3
    cum = -torch.rand(batch * beams, device="cuda")
    st = torch.cuda.Stream()
    o, w = outs(), outs()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        beam.select(x, cum, None, *o, batch, beams, V, n)  # the stream's workspace
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        beam.select(x, cum, None, *o, batch, beams, V, n)
    for rep in range(4):
        x.copy_(torch.randn_like(x) * 3)
        for t in o:
            t.fill_(0)
        g.replay()
        beam.select(x, cum, None, *w, batch, beams, V, n)  # eager, on the current stream, at the same time
        torch.cuda.synchronize()
        for a, b in zip(o, w):
            assert torch.equal(a, b), rep


def test_captures_are_told_apart(beam):
    import torch
    from helios_glm53flash_amd._lib import lib
    st, side = torch.cuda.Stream(), torch.cuda.Stream()
    x = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    ids = []
    for _ in range(4):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            side.wait_stream(st)
            with torch.cuda.stream(side):
                x.add_(1)
            ids.append(lib.hx_capture_id(st.cuda_stream))
            assert lib.hx_capture_id(side.cuda_stream) == ids[-1]
            st.wait_stream(side)
        assert lib.hx_capture_id(st.cuda_stream) == 0 and lib.hx_capture_id(None) == 0
        del g
    assert 0 not in ids and len(set(ids)) == 4


def test_calls_of_two_captures_on_one_stream(beam):
    """Calls of a capture share memory of its graph, small ones first, with other tensors made and dropped between them; two graphs
    of one stream replay in any order, beside eager calls."""
    import torch
    from helios_glm53flash_amd import w4
    K, N, group = 4096, 256, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    q = torch.randint(0, 16, (N, K), generator=gen, device="cuda").to(torch.uint8)
    w = w4.W4Words(w4.pack(q), torch.full((N, K // group), 0.125, dtype=torch.float16, device="cuda"), None, K, group)
    batch, beams, n = 2, 4, 8
    cum = -torch.rand(batch * beams, device="cuda")
    st = torch.cuda.Stream()
    graphs = []

    def calls(x, y, logits, outs):
        for M in (16, 64, 16):
            w4.gemm(y[M], x, w, M, N, K, True)
            torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
            beam.select(logits, cum, None, *outs, batch, beams, 50000, n)

    for g in range(2):
        x = torch.randn((64, K), device="cuda").half()
        y = {M: torch.zeros((M, N), device="cuda") for M in (16, 64)}
        logits = torch.randn((batch * beams, 50000), device="cuda")
        outs = [torch.zeros((batch, n), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            calls(x, y, logits, outs)
        graphs.append((graph, x, y, logits, outs))
    for rep in range(6):
        graph, x, y, logits, outs = graphs[(0, 1, 1, 0, 1, 0)[rep]]
        x.copy_(torch.randn_like(x))
        logits.copy_(torch.randn_like(logits) * 3)
        torch.cuda.synchronize()
        graph.replay()
        want_y = {M: torch.empty((M, N), device="cuda") for M in (16, 64)}
        want = [torch.empty_like(o) for o in outs]
        calls(x, want_y, logits, want)
        torch.cuda.synchronize()
        assert all(torch.equal(y[M], want_y[M]) for M in y) and all(torch.equal(a, b) for a, b in zip(outs, want)), rep


def test_select_on_a_forked_stream_of_a_capture(beam):
    """A captured call on a stream that was forked from the capturing one depends on no workspace of that stream."""
    import torch
    batch, beams, V, n = 2, 4, 20000, 8
    x = torch.randn((batch * beams, V), device="cuda") * 3
    cum = -torch.rand(batch * beams, device="cuda")
    outs = [[torch.empty((batch, n), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64)]
            for _ in range(3)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        beam.select(x, cum, None, *outs[0], batch, beams, V, n, stream=side)
        beam.select(x, cum, None, *outs[1], batch, beams, V, n)
        here.wait_stream(side)
    for rep in range(4):
        x.copy_(torch.randn_like(x) * 3)
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(side):
            beam.select(x, cum, None, *outs[2], batch, beams, V, n)
        torch.cuda.synchronize()
        for a, b, c in zip(*outs):
            assert torch.equal(a, c) and torch.equal(b, c), rep


@pytest.mark.parametrize("batch,beams,V,n", [(1, 4, 20001, 8), (3, 1, 5, 128), (600, 1, 9000, 3), (2, 300, 5000, 33)])
def test_select_in_a_workspace_of_the_least_size(beam, batch, beams, V, n):
    import torch
    from helios_glm53flash_amd._lib import lib
    x = torch.randn((batch * beams, V), device="cuda")
    cum = -torch.rand(batch * beams, device="cuda")
    want = [torch.empty((batch, n), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64)]
    beam.select(x, cum, None, *want, batch, beams, V, n)
    need = lib.hx_beam_select_workspace_size(batch, beams, V, n)
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    ws[:65536].zero_()
    for _ in range(3):
        got = [torch.empty_like(o) for o in want]
        assert lib.hx_beam_select(x.data_ptr(), cum.data_ptr(), None, *(o.data_ptr() for o in got), batch, beams, V, n, V, 0, 1,
                                  torch.cuda.current_stream().cuda_stream, ws.data_ptr(), need) == 0
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool((ws[need:] == 0x5A).all()) and bool((ws[:65536] == 0).all())


def test_select_leaves_the_counters_zero(beam):
    import torch
    from helios_glm53flash_amd import exl3
    x = torch.randn((64, 9000), device="cuda")
    cum = torch.zeros(64, device="cuda")
    for batch, n in ((64, 4), (1, 128), (16, 16)):
        o = [torch.empty((batch, n), dtype=d, device="cuda") for d in (torch.float32, torch.int64, torch.int64)]
        beam.select(x, cum, None, *o, batch, 64 // batch, 9000, n)
        ws = exl3.workspace(0, x.device)
        assert int(ws[:65536].view(torch.int32).abs().sum()) == 0


# ------------------------------------------------------------------ states

@pytest.mark.parametrize("shape,dim", [((12, 7), 0), ((12,), 0), ((3, 12, 5, 16), 1), ((2, 3, 12, 4, 8), 2), ((5, 12), 1),
                                       ((12, 1, 1), 0), ((1, 12, 33), -2)])
@pytest.mark.parametrize("dtype", ["float16", "float32", "uint8", "int64", "bool", "bfloat16"])
def test_reorder(beam, shape, dim, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    src = torch.randint(0, 2 if dtype == "bool" else 100, shape, generator=g, device="cuda").to(dt)
    batch, beams = 3, 4
    for out in (1, 4, 6):
        parents = torch.randint(0, beams, (batch, out), generator=g, device="cuda")
        d = list(shape)
        d[dim] = batch * out
        dst = torch.zeros(d, dtype=dt, device="cuda")
        beam.reorder(src, parents, dst, batch, beams, out, dim=dim)
        at = (torch.arange(batch, device="cuda")[:, None] * beams + parents).view(-1)
        assert torch.equal(dst, src.index_select(dim, at))


@pytest.mark.parametrize("tokens,width", [(1, 8), (37, 24), (100, 13), (128, 576)])
def test_reorder_of_a_cache_below_its_capacity(beam, tokens, width):
    """Views of a cache [layers][rows][heads][capacity][width] and [layers][rows][capacity][width]: only the filled part is
    written, rows with parents outside the beams are left as they were."""
    import torch
    cap, batch, beams = 128, 2, 3
    cache = torch.randn((2, 4, batch * beams, cap, width), device="cuda").half()
    parents = torch.tensor([[2, 2, 0], [-1, 1, 3]], device="cuda")
    src, out = cache[0], torch.full_like(cache[1], 5.0)
    beam.reorder(src[:, :, :tokens], parents, out[:, :, :tokens], batch, beams, beams, dim=1)
    want = torch.full_like(out, 5.0)
    for r, s in enumerate((2, 2, 0, None, 4, None)):
        if s is not None:
            want[:, r, :tokens] = src[:, s, :tokens]
    assert torch.equal(out, want)
    heads = torch.randn((batch * beams, 5, cap, width), device="cuda").half()
    out = torch.zeros_like(heads)
    beam.reorder(heads[:, :, :tokens], parents, out[:, :, :tokens], batch, beams, beams)
    assert torch.equal(out[0], torch.cat([heads[2][:, :tokens], torch.zeros_like(heads[2][:, tokens:])], dim=1))


def test_reorder_unaligned_and_large(beam):
    import torch
    raw = torch.randint(0, 255, (2, 6 * 1003 + 16), device="cuda").to(torch.uint8)
    for off in (0, 1, 2, 4, 8):
        src = raw[0][off:off + 6 * 1003].view(6, 1003)
        for doff in (0, 3, 4):
            dst = raw[1][doff:doff + 6 * 1003].view(6, 1003)
            p = torch.tensor([[1, 1, 0], [2, 0, 2]], device="cuda")
            beam.reorder(src, p, dst, 2, 3, 3)
            assert torch.equal(dst, src[[1, 1, 0, 5, 3, 5]])
    for width in (300_000, 1_000_003):  # few large pieces, each in parts
        src = torch.randint(0, 255, (6, width), device="cuda").to(torch.uint8)
        dst = torch.full((8, width), 255, dtype=torch.uint8, device="cuda")
        beam.reorder(src, p, dst[1:-1], 2, 3, 3)
        assert torch.equal(dst[1:-1], src[[1, 1, 0, 5, 3, 5]])
        assert bool((dst[0] == 255).all()) and bool((dst[-1] == 255).all())
    big = torch.zeros((3, (1 << 31) + 48), dtype=torch.uint8, device="cuda")  # offsets past 2^32 bytes
    big[2, -100:] = torch.arange(100, dtype=torch.uint8, device="cuda")
    big[1, -1] = 9
    dst = torch.ones_like(big)
    beam.reorder(big, torch.tensor([[2, 0, 2]], device="cuda"), dst, 1, 3, 3)
    assert torch.equal(dst[0], big[2]) and torch.equal(dst[1], big[0]) and torch.equal(dst[2], big[2])


def test_reorder_refusals(beam):
    import torch
    from helios_glm53flash_amd._lib import HxError
    x = torch.zeros((6, 8), device="cuda")
    p = torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    with pytest.raises(HxError, match="overlap"):
        beam.reorder(x, p, x, 2, 3, 3)
    with pytest.raises(HxError, match="overlap"):
        beam.reorder(torch.zeros_like(x), p, torch.zeros((1, 8), device="cuda").expand(6, 8), 2, 3, 3)
    with pytest.raises(ValueError, match="reduce"):
        big = torch.zeros((6, 4, 5, 8), device="cuda")
        beam.reorder(big[:, :3, :3, :6], p, torch.zeros((6, 3, 3, 6), device="cuda"), 2, 3, 3)
    with pytest.raises(ValueError):
        beam.reorder(x, p, torch.zeros((5, 8), device="cuda"), 2, 3, 3)
    with pytest.raises(ValueError):
        beam.reorder(x, p, torch.zeros((6, 8), device="cuda").half(), 2, 3, 3)
    # a broadcast source is an ordinary one
    dst = torch.zeros_like(x)
    beam.reorder(torch.arange(8.0, device="cuda").expand(6, 8), p, dst, 2, 3, 3)
    assert torch.equal(dst, torch.arange(8.0, device="cuda").expand(6, 8))


def test_decode_steps_of_a_small_model(beam):
    """Beam search over a small model as a serving loop runs it: the 4-bit head's rows as embedding, a MoE layer, the state
    of each beam, the head's logits, selection, reordering; each call's result against 64 bits on the call's own inputs."""
    import torch
    from helios_glm53flash_amd import moe, w4
    V, K, group, batch, beams, n, eos = 3001, 256, 64, 2, 4, 8, 5
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    q = (torch.randn((V, K), generator=g, device="cuda") * 2.5 + 8).round().clamp(0, 15).to(torch.uint8)
    sc = ((0.5 + torch.rand((V, K // group), generator=g, device="cuda")) * 0.4 / K ** 0.5).half()
    head = w4.W4Words(w4.pack(q), sc, None, K, group)
    W = (q.double() - 8) * sc.double().repeat_interleave(group, dim=1)
    layer = moe.MoeLayer(moe.ExpertSet.synthetic(16, K, 128, 2, seed=1), moe.synthetic_dense_mlp(K, 128, 2, seed=2), topk=4)
    rows = batch * beams
    cum = torch.full((batch, beams), float("-inf"), device="cuda")
    cum[:, 0] = 0.0
    done = torch.zeros((batch, beams), dtype=torch.uint8, device="cuda")
    tokens = torch.full((batch, beams), 17, dtype=torch.int64, device="cuda")
    state = torch.zeros((2, rows, 6, K), dtype=torch.float16, device="cuda")  # ping-pong cache of hidden states
    h = torch.empty((rows, K), dtype=torch.float16, device="cuda")
    logits = torch.empty((rows, V), device="cuda")
    scores = torch.empty((batch, n), device="cuda")
    parents, toks = (torch.empty((batch, n), dtype=torch.int64, device="cuda") for _ in range(2))
    for step in range(5):
        w4.embed(head, tokens.view(-1), h, rows, K ** 0.5)
        assert torch.equal(h, (W[tokens.view(-1)] * K ** 0.5).half())
        y = layer(h, torch.randn((rows, 16), generator=g, device="cuda").half())
        x = (h.float() + y.float() / y.float().abs().amax().clamp(min=1e-6)).half()
        src, dst = state[step % 2], state[(step + 1) % 2]
        src[:, step] = x
        w4.gemm(logits, x, head, rows, V, K, True)
        ref = x.double() @ W.T
        assert bool(((logits.double() - ref).abs() <= (K + 8) * 2.0 ** -24 * (x.double().abs() @ W.abs().T)).all())
        logits[:, 3] = float("-inf")
        s, p, t = check(beam, logits, cum.view(-1).cpu().numpy(), done.view(-1).cpu().numpy(), batch, beams, V, n, eos)
        beam.select(logits, cum.view(-1), done.view(-1), scores, parents, toks, batch, beams, V, n, eos)
        keep = parents[:, :beams].contiguous()
        assert bool((keep >= 0).all()) and np.array_equal(keep.cpu().numpy(), p[:, :beams])
        beam.reorder(src[:, :step + 1], keep, dst[:, :step + 1], batch, beams, beams)
        at = (torch.arange(batch, device="cuda")[:, None] * beams + keep).view(-1)
        assert torch.equal(dst[:, :step + 1], src[at][:, :step + 1])
        cum, tokens = scores[:, :beams].contiguous(), toks[:, :beams].contiguous()
        new_done = torch.empty_like(done)
        beam.reorder(done.view(-1), keep, new_done.view(-1), batch, beams, beams)
        done = new_done | (tokens == eos).to(torch.uint8)
        if step == 1:
            done[0, 1] = 1
