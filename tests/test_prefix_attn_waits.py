"""What the blocks of `shared_prefix_attention` do when a wait runs out, on the
CPU: the order of waits and barriers is read from the kernel's source and run
as a small machine, with every choice of which warp gives up at which wait."""

import itertools
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "epic-kernel_b200" / "csrc" / "ek_prefix_attn.cu").read_text()
WARPS = 4  # of a softmax warpgroup


def softmax_loop():
    """The tile loop of a softmax warp of many_rows, as (operations of a tile, loop condition)."""
    kernel = SOURCE[SOURCE.index("many_rows(const __grid_constant__") :]
    start = kernel.index("for (int use = 0;")
    body = kernel[start : kernel.index("wait(p_empty + w, (mine - 1) & 1)", start)]
    condition = re.match(r"for \(int use = 0; ([^;]*);", body).group(1)
    operations = []
    pattern = (r"if \(!\(ok = agree\(ok\)\)\) break;|^\s*sync\(\);|"
               r"if \((?:use > 0 && )?!\(ok = spin\((\w+) \+ w, [^;]*\)\)\) (break|continue);")
    for m in re.finditer(pattern, body, re.M):
        if "agree" in m.group(0):
            operations.append(("vote",))
        elif "sync" in m.group(0):
            operations.append(("sync",))
        else:
            operations.append(("wait", m.group(1), m.group(2), "use > 0" in m.group(0)))
    return operations, condition


def warp(operations, condition, tiles, gives_up):
    """A softmax warp with 8-bit rows; its wait number `gives_up` runs out (None: none). Yields (barrier, count, ok)."""
    ok, waits, use = True, 0, 0
    while use < tiles and ("ok" not in condition or "I8" in condition or ok):
        leave = False
        for op in operations:
            if op[0] == "wait":
                if op[3] and use == 0:
                    continue
                ok = waits != gives_up
                waits += 1
                if not ok:
                    leave = op[2] == "break"
                    break
            else:
                everyone = yield ("group", WARPS, ok)
                if op[0] == "vote":
                    ok = everyone
                    if not ok:
                        leave = True
                        break
        if leave:
            break
        use += 1
    yield ("block", 2 * WARPS, ok)
    return


def run(warps):
    """Runs [(group, warp), ...] until all have ended; False if some stand at a barrier that never fills."""
    at = {}
    for i, (_, w) in enumerate(warps):
        at[i] = next(w)
    while at:
        moved = False
        for key in {(b, warps[i][0] if b == "group" else None) for i, (b, _, _) in at.items()}:
            here = [i for i, (b, _, _) in at.items() if (b, warps[i][0] if b == "group" else None) == key]
            if len(here) < at[here[0]][1]:
                continue
            moved = True
            everyone = all(at[i][2] for i in here)
            for i in here:
                try:
                    at[i] = warps[i][1].send(everyone)
                except StopIteration:
                    del at[i]
        if not moved:
            return False
    return True


def test_the_loop_is_read():
    operations, _ = softmax_loop()
    kinds = [op[0] for op in operations]
    assert kinds.count("wait") == 3 and [op[1] for op in operations if op[0] == "wait"] == ["s_full", "p_empty", "p_empty"]
    assert kinds.count("vote") + kinds.count("sync") == 2 and "wait" not in kinds[:2]


@pytest.mark.parametrize("tiles", [(1, 1), (2, 1), (2, 2), (3, 3), (4, 3)])
@pytest.mark.parametrize("idle", [False, True])
def test_softmax_warps_meet_at_their_barriers(tiles, idle):
    """Whichever wait of a warp runs out, no warp is left at a barrier of the warpgroup or of the block. A warp without
    rows takes the other wait for p_empty."""
    operations, condition = softmax_loop()
    waits = [i for i, op in enumerate(operations) if op[0] == "wait"]
    drop = waits[1] if not idle else waits[2]
    operations = [op for i, op in enumerate(operations) if i != drop]
    points = [None, *range(2 * max(tiles) - 1)]
    for first in itertools.product(points, repeat=WARPS):
        warps = [(0, warp(operations, condition, tiles[0], p)) for p in first]
        warps += [(1, warp(operations, condition, tiles[1], first[0] if tiles[1] > 1 else None)) for _ in range(WARPS)]
        assert run(warps), f"warps that give up at {first} leave others at a barrier"


def loader_part(kernel, begin):
    text = SOURCE[SOURCE.index(kernel + "(const __grid_constant__") :]
    text = text[text.index(begin) :]
    return text[: text.index("} else ")]


def in_flight_at_the_end(steps, stages, fails_at, only_if_gave_up):
    """Copies that may still be landing when a block's threads meet after its consumers gave up waiting for copy
    `fails_at`: the loader issues while a buffer is free and waits for the last copy of each buffer, always or only if
    it could not issue them all."""
    issued = min(steps, fails_at + stages)
    waited = range(max(0, issued - stages), issued) if issued < steps or not only_if_gave_up else ()
    return [n for n in range(fails_at, issued) if n not in waited]


@pytest.mark.parametrize("kernel,begin", [("few_rows", "if (warp == kWarps) {"), ("many_rows", "if (warp == C::LOADER) {")])
def test_no_copy_is_in_flight_when_the_shared_memory_is_used_again(kernel, begin):
    part = loader_part(kernel, begin)
    assert part.count("&quiet") >= 1, "the loader waits for its copies, whatever the state of the block"
    drain = part[: part.index("int quiet")]
    only_if_gave_up = re.search(r"if \(n < (steps|items)\) \{[^}]*$", drain) is not None
    for steps, stages in itertools.product(range(1, 9), range(1, 5)):
        for fails_at in range(steps):
            assert not in_flight_at_the_end(steps, stages, fails_at, only_if_gave_up), (steps, stages, fails_at)


def test_rows_are_staged_only_if_no_softmax_warp_gave_up():
    """O goes to global memory through the memory of K and V tiles, which hold late copies if a wait has run out."""
    kernel = SOURCE[SOURCE.index("many_rows(const __grid_constant__") :]
    end = kernel[kernel.index("wait(p_empty + w, (mine - 1) & 1)") : kernel.index("bulk_store(")]
    assert re.search(r"ok = ek::barrier_all<3, 256>\(ok\);.*if \(!ok\) m = NAN, l = NAN;.*if \(mine > 0 && ok\)", end, re.S)
