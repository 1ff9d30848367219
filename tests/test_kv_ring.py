"""The ring of key and value tiles that the tcgen05 attention kernels share: whether every wait for a tile can only pass once that tile has landed.

A tile's barrier says the parity of the phases it has completed, so a wait passes both when its own phase is over and while the phase before it is not.  The model below walks through
every order in which loads may land and the three warps (loads, Q K^T, P V) may go on, with the kernels' rules for when each does."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "tile-rs_b200" / "csrc"


def tiles(segments):
    """(kind, step) in the order they are loaded: K_0, K_1, V_0, K_2, V_1, ..., K_{n-1}, V_{n-2}, V_{n-1} of every segment; steps count on."""
    order, before = [], 0
    for n in segments:
        order.append(("k", before))
        for j in range(n - 1):
            order += [("k", before + j + 1), ("v", before + j)]
        order.append(("v", before + n - 1))
        before += n
    return order


def false_passes(segments, ring, p_first, ahead=True):
    """Tiles for which a wait can pass before they have landed.  p_first: P V waits for its probabilities before it waits for V.  ahead: Q K^T of step s waits for the P V of s - 2."""
    order, steps = tiles(segments), sum(segments)
    at = {t: i for i, t in enumerate(order)}
    wrong, seen, todo = set(), set(), [(0, 0, 0, 0, False)]
    # landed: a bit a tile (loads may land in any order); issued: tiles asked for; qk, pv: steps whose products are issued; waited: P V has passed its first wait of step pv
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        issued, landed, qk, pv, waited = state

        def passes(i):  # a wait for tile i: completed phases of its slot are those of the slot's tiles that have landed
            done = sum(1 for t in range(i % ring, issued, ring) if landed >> t & 1)
            return (done & 1) != (i // ring & 1)

        def used(i):
            kind, s = order[i]
            return s < (qk if kind == "k" else pv)

        if issued < len(order) and (issued < ring or used(issued - ring)):
            todo.append((issued + 1, landed, qk, pv, waited))
        for i in range(issued):
            if not landed >> i & 1:
                todo.append((issued, landed | 1 << i, qk, pv, waited))
        if qk < steps and (not ahead or qk < 2 or pv >= qk - 1):
            # S of the step before has been read once its softmax is through, which nothing else holds up
            i = at["k", qk]
            if passes(i):
                if not (i < issued and landed >> i & 1):
                    wrong.add(order[i])
                else:
                    todo.append((issued, landed, qk + 1, pv, waited))
        if pv < steps:
            i = at["v", pv]
            probabilities = qk > pv
            if p_first:
                if probabilities and passes(i):
                    if not (i < issued and landed >> i & 1):
                        wrong.add(order[i])
                    else:
                        todo.append((issued, landed, qk, pv + 1, False))
            elif not waited:
                if passes(i):
                    if not (i < issued and landed >> i & 1):
                        wrong.add(order[i])
                    else:
                        todo.append((issued, landed, qk, pv, True))
            elif probabilities:
                todo.append((issued, landed, qk, pv + 1, False))
    return wrong


SEGMENTS = [(1,), (2,), (3,), (6,), (1, 1, 1, 1), (1, 3, 1, 2), (2, 2, 2), (3, 1, 3), (4, 4)]


@pytest.mark.parametrize("segments", SEGMENTS)
def test_values_after_probabilities_in_a_ring_of_three(segments):
    assert not false_passes(segments, 3, p_first=True)


def test_values_before_probabilities_are_unsafe_in_a_ring_of_three():
    """The model finds the order that a slow load makes wrong: V_2 takes the slot that K_2 has not reached yet."""
    assert ("v", 2) in false_passes((6,), 3, p_first=False)


@pytest.mark.parametrize("ring", [4, 5, 6, 8])
@pytest.mark.parametrize("segments", SEGMENTS)
def test_longer_rings_in_either_order(segments, ring):
    assert not false_passes(segments, ring, p_first=False)


def test_the_kernels_with_a_ring_of_three_wait_in_that_order():
    for name, p_wait, v_wait in (("attention_tc.cuh", r"wait_p\(0, j\)", r"wait_kv\(v_pos\(j\)\)"), ("attention_paged_tc.cuh", r"p_ready\[g\], \(done", r"wait_kv\(v_pos\(j\)")):
        text = re.sub(r"//.*", "", (CSRC / name).read_text())
        assert re.search(p_wait, text).start() < re.search(v_wait, text).start(), name
