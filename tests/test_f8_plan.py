"""Which kernel takes a call of the 8-bit linear and its gated pair (csrc/hx_f8_plan.hpp, compiled for the host), and its workspace."""
import ctypes as C
import itertools
import random
import shutil
import subprocess
from pathlib import Path

import pytest

import test_gpu_f8 as gpu
from test_gpu_f8_tiles import EXACT, FAST, GATED, TILES, TILES2

ROOT = Path(__file__).resolve().parent.parent
KINDS = ["rows", "64x32", "64x64", "128x64", "128x128", "256x32", "256x64", "256x256", "none"]
COUNTERS = 64 * 1024


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no C++ compiler")
    so = tmp_path_factory.mktemp("plan") / "f8_plan.so"
    subprocess.run([cxx, "-std=c++20", "-O1", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{ROOT / 'helios_glm53flash_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cpp" / "f8_plan.cpp"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.f8_call_workspace.restype = C.c_size_t
    return lib


def plan(lib, M, K, N, sums, split=True):
    out = (C.c_long * 6)()
    lib.f8_plan(M, N, K, sums, int(split), out)
    return dict(zip(("kind", "splits", "steps", "tiles", "partial", "products"), (KINDS[out[0]], *out[1:])))


def tiles(lib):
    """(sums, kind): rows, columns, whether K may be split."""
    t = {}
    for sums, kind in itertools.product(range(3), range(1, 8)):
        out = (C.c_int * 3)()
        lib.f8_tile(sums, kind, out)
        if out[0]:
            t[sums, KINDS[kind]] = (out[0], out[1], bool(out[2]))
    return t


def need(p):
    return COUNTERS + p["partial"] + p["products"] if p["partial"] or p["products"] else 0


def test_sizes_of_the_gpu_tests_reach_what_they_name(lib):
    for (sums, kind, splits), (M, K, N) in [*TILES.items(), *TILES2.items()]:
        p = plan(lib, M, K, N, sums)
        assert (p["kind"], p["splits"]) == (kind, splits), (sums, kind, splits, p)
        assert K % 128 and N % 128
    for sums, kind, _ in TILES2:
        assert TILES2[sums, kind, 1][2] % 256 > 128


def test_every_kernel_has_a_size(lib):
    """Whole, and where K may be split, in parts of each number that some call of up to 4000 rows, K up to 12800 and N up to 20000 has."""
    t = tiles(lib)
    assert len(t) == 5 + 4 + 6 and {(s, k) for s, k, _ in TILES} == set(t)
    for (sums, kind), (_, _, split) in t.items():
        assert (sums, kind, 1) in TILES
        assert split == any(s > 1 for a, b, s in TILES if (a, b) == (sums, kind))
    r, seen = random.Random(0), set()
    for _ in range(60000):
        sums = r.randrange(3)
        M, K, N = int(9 * 444 ** r.random()), 16 * int(800 ** r.random()), int(16 * 1250 ** r.random())
        p = plan(lib, M, K, N // 16 * 16 if sums == GATED else N, sums)
        seen.add((sums, p["kind"], p["splits"]))
    assert len(seen) > 45 and seen <= set(TILES), seen - set(TILES)


def test_few_rows(lib):
    for M, K, N in itertools.product((1, 8), (16, 4096, 4112, 16384), (1, 4096, 151552)):
        assert plan(lib, M, K, N, EXACT)["kind"] == "rows"
    for M, K, N in gpu.GSHAPES:
        assert (plan(lib, M, K, N, GATED)["kind"] == "rows") == (M <= 8)


EXTREME = list(itertools.product((1, 8, 9, 300, 1 << 22, (1 << 30) + 5, (1 << 31) - 1), (16, 144, 4096, 65536, 1 << 22), (16, 4096, 151552, (1 << 28) - 16, 1 << 28)))


@pytest.mark.parametrize("sums", [FAST, EXACT, GATED])
def test_every_call_has_a_kernel_and_fits_its_bounds(lib, sums):
    """Launches of a call within their limits; counters and bytes of a workspace within what they are sized for."""
    t = tiles(lib)
    for M, K, N in EXTREME:
        most = lib.f8_most_rows(N, sums == GATED)
        assert most > 0 and most % 256 == 0
        want = 0
        for rows in {min(M, most), M % most or most if M > most else M}:
            for split in (True, False):
                p = plan(lib, rows, K, N, sums, split)
                assert p["kind"] != "none", (M, K, N)
                kb = -(-K // 128)
                assert (p["splits"] - 1) * p["steps"] < kb <= p["splits"] * p["steps"]
                assert split or p["splits"] == 1
                if split:
                    want = max(want, need(p))
                if p["kind"] == "rows":
                    assert rows <= 8
                    continue
                bn, bm, _ = t[sums, p["kind"]]
                mt, nt = -(-rows // bm), -(-(2 * N if sums == GATED else N) // bn)
                assert p["tiles"] == mt * nt <= 1 << 22
                arrivals = (mt * nt if need(p) else 0) + (mt * -(-N // 128) if p["products"] else 0)  # of the parts of K, then of the blocks of outputs
                assert 4 * arrivals <= COUNTERS
                assert need(p) <= COUNTERS + (64 << 20)
        assert lib.f8_call_workspace(M, N, K, sums) == want, (M, K, N)


def test_workspace_of_the_library(lib):
    """The exported sizes are the plan's: of the linear the larger of its two ways."""
    from helios_glm53flash_amd import _lib
    for M, K, N in [*TILES.values(), (1, 4096, 2048), (8, 16384, 4096), ((1 << 30) + 5, 16, 16), (5, 4096, 1 << 28)]:
        size = max(lib.f8_call_workspace(M, N, K, sums) for sums in (FAST, EXACT))
        assert _lib.lib.hx_f8_gemm_workspace_size(M, N, K) == size
        if N % 16 == 0:
            assert _lib.lib.hx_f8_gate_up_workspace_size(M, N, K) == lib.f8_call_workspace(M, N, K, GATED)
    assert _lib.lib.hx_f8_gate_up_workspace_size((1 << 30) + 5, 16, 16) > 0  # of the five rows behind the first launch
