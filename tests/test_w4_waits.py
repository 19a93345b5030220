"""The LDS ring of the 4-bit linear's tiles in the compiled code: at the barrier ahead of a step, the loads into LDS of that and
all earlier steps are complete on every path, whatever order the compiler gave the loads (the waits count them)."""
import re

import pytest

import test_mfma_waits as waits


def follow(bb, entry, na):
    """Follows every path from `entry`: (loads that may be late, loads outstanding) at the first barrier at fault, or None.
    Every step issues `na` loads into LDS, so step b's barrier may find those of later steps outstanding only."""
    todo, seen = [(entry, (), 0)], set()
    while todo:  # block, outstanding ops (oldest first), loads into LDS issued less those due by now
        k, out, spare = todo.pop()
        if (k, out, spare) in seen:
            continue
        seen.add((k, out, spare))
        for op in bb[k][0]:
            if op in ("A", "V"):
                out = (out + (op,))[-63:]
                spare += op == "A"
            elif op == "B":
                spare = max(0, spare - na)  # behind the last step the barriers go on and nothing is due
                if out.count("A") > spare:
                    return spare, out.count("A")
            else:
                out = out[len(out) - op:] if op < len(out) else out
        todo += [(s, out, spare) for s in bb[k][1]]
    return None


@pytest.mark.skipif(not (waits.LLVM / "llvm-objdump").exists(), reason="no llvm-objdump")
def test_every_step_is_complete_at_its_barrier(tmp_path, monkeypatch):
    if not waits.LIB.exists():
        import __graft_entry__
        __graft_entry__.build()
    monkeypatch.setattr(waits, "KERNELS", ("w4_tile_kernel",))
    kernels = waits.tile_kernels(waits.LIB, tmp_path)
    # six tiles, three group classes, with and without zero points; three tiles for groups loaded one by one
    assert len(kernels) == 6 * 3 * 2 + 3 * 2 * 2
    for name, bb in kernels.items():
        bm = int(re.search(r"w4_tile_kernelILi(\d+)E", name).group(1))
        first = min(bb)
        todo, reach = [first], set()
        while todo:
            k = todo.pop()
            if k not in reach:
                reach.add(k)
                todo += bb[k][1]
        assert sum(ops.count("A") for k, (ops, _) in bb.items() if k in reach) >= 2 * bm // 16, name
        assert follow(bb, first, bm // 16) is None, f"{name}: {follow(bb, first, bm // 16)}"


@pytest.mark.parametrize("loop,ok", [(["B", "A", "V", 4], True), (["B", "A", "V", 5], True), (["B", "A", "V", 6], False)])
def test_checker_on_a_ring_of_three(loop, ok):
    """Two steps of one load into LDS and one other ahead: a wait for 4 (or 5: the late one is no load into LDS) outstanding
    leaves the next step's complete, one for 6 does not."""
    bb = {0: (["A", "V", "A", "V", "A", "V", loop[-1]], [1]), 1: (loop, [1, 2]), 2: ([0, "B"], [])}
    assert (follow(bb, 0, 1) is None) == ok
