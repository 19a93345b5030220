"""The LDS ring of the 8-bit linear's tiles in the compiled code: at the barrier ahead of a step, the loads into LDS of that and
all earlier steps are complete on every path, whatever order the compiler gave the loads (the waits count them)."""
import re

import pytest

import test_mfma_waits as waits


def ring(name):
    """Loads into LDS of a wave that loads: of scales ahead of the first step; a step's (scales, x, weights); steps ahead."""
    wn, wm, tn, tm, ahead = map(int, re.search(r"f8_tile_kernel" + 5 * r"\w*?Li(\d+)E", name).groups())
    loaders = 4 if wn * wm == 8 else wn * wm
    return 2 * -(-wm * tm // loaders), 1 + (wm * tm + wn * tn) * 2 // loaders, ahead - 1


def loading(bb):
    """The paths of a wave that loads: a branch around loads into LDS is not taken."""
    out = {}
    for k, (ops, succ) in bb.items():
        loads = [s for s in succ if "A" in bb[s][0] and "B" not in bb[s][0] and set(succ) - {s} == set(bb[s][1])]
        out[k] = (ops, loads or succ)
    return out


def follow(bb, entry, scales, step, ahead):
    """Follows every path from `entry` on which a wave has issued all loads ahead of the first step: (loads that may be late, loads
    outstanding) at the first barrier at fault, None if there is none, or "no barrier"."""
    todo, seen, met = [(entry, (), 0, False)], set(), False
    while todo:  # block, outstanding ops (oldest first), loads issued less those due by now, behind the first barrier
        k, out, spare, begun = todo.pop()
        if (k, out, spare, begun) in seen:
            continue
        seen.add((k, out, spare, begun))
        for op in bb[k][0]:
            if op in ("A", "V"):
                out = (out + (op,))[-63:]
                spare += op == "A"
            elif op == "B":
                if not begun:
                    if spare != scales + ahead * step:
                        break
                    spare -= scales
                begun = met = True
                spare = max(0, spare - step)  # behind the last step the barriers go on and nothing is due
                if out.count("A") > spare:
                    return spare, out.count("A")
            else:
                out = out[len(out) - op:] if op < len(out) else out
        else:
            todo += [(s, out, spare, begun) for s in bb[k][1]]
    return None if met else "no barrier"


@pytest.mark.skipif(not (waits.LLVM / "llvm-objdump").exists(), reason="no llvm-objdump")
def test_every_step_is_complete_at_its_barrier(tmp_path, monkeypatch):
    if not waits.LIB.exists():
        import __graft_entry__
        __graft_entry__.build()
    monkeypatch.setattr(waits, "KERNELS", ("f8_tile_kernel",))
    kernels = waits.tile_kernels(waits.LIB, tmp_path)
    assert len(kernels) == 5 + 4 + 6  # fp16 outputs, fp32 outputs, gated pair
    for name, bb in kernels.items():
        fault = follow(loading(bb), min(bb), *ring(name))
        assert fault is None, f"{name}: {fault}"


STEP = ["A", "A", "V"]


@pytest.mark.parametrize("late,fault", [(3, None), (4, None), (5, (2, 3))])
def test_checker_on_a_ring_of_three(late, fault):
    """Two steps of two loads ahead, one of scales before them: a wait for 3 (or 4: the late ones of the step due
    are no loads into LDS) outstanding leaves the next step's complete, one for 5 does not."""
    bb = {0: (["A"] + STEP + STEP + [late], [1]), 1: (["B"] + STEP + [late], [1, 2]), 2: ([0, "B"], [])}
    assert follow(bb, 0, 1, 2, 2) == fault


def test_checker_on_a_branch_around_the_loads():
    bb = {0: (["A"] + STEP, [1]), 1: ([0, "B"], [2, 3]), 2: (STEP, [3]), 3: ([], [1, 4]), 4: ([0, "B"], [])}
    assert loading(bb)[1][1] == [2] and follow(loading(bb), 0, 1, 2, 1) is None
    late = {**bb, 1: ([1, "B"], [2, 3])}
    assert follow(loading(late), 0, 1, 2, 1) is None  # the one that may be late is none of LDS
    assert follow(loading({**bb, 1: ([2, "B"], [2, 3])}), 0, 1, 2, 1) == (0, 1)
    assert follow({0: (["A"], [1]), 1: ([0, "B"], [])}, 0, 1, 2, 1) == "no barrier"
