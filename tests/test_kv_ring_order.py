"""Every place where the tcgen05 attention kernels with a ring of three tiles wait for values: behind the wait for probabilities of the same step and query tile (tests/test_kv_ring.py has the reason)."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "tile-rs_b200" / "csrc"


def source(name):
    return re.sub(r"\s+", " ", re.sub(r"//.*", "", (CSRC / name).read_text()))


def in_order_tc(text):
    """Two places, one to a query tile.  The first has the step's probabilities before it in the same condition; so has the second, which waits for values only where the first tile has no such step."""
    first = text.find("if (!(ok = wait_p(0, j) && wait_kv(v_pos(j)))) break; issue_pv(0,")
    second = text.find("if (!(ok = wait_p(1, j) && (j < n_a || wait_kv(v_pos(j))))) break; issue_pv(1,")
    return text.count("wait_kv(v_pos(j)") == 2 and 0 <= first < second and "if (j < n_a) { if (!(ok = wait_p(0, j)" in text


def in_order_paged(text):
    """One place, in the loop over query tiles, straight behind that tile's wait for probabilities and only while the step's values have not been waited for."""
    at = re.search(r"bool landed = false; for \(int g = 0; g < 2 && ok; \+\+g\) \{ if \(j >= n_of\[g\]\) continue;.*?"
                   r"ok = __all_sync\(0xffffffffu, ptx::mbar_wait\(&bars->p_ready\[g\], \(done\[g\] \+ j\) & 1u, abort_flag, p\.status, 162 \+ g\)\); "
                   r"if \(ok && !landed\) ok = landed = wait_kv\(v_pos\(j\)", text)
    return text.count("wait_kv(v_pos(j)") == 1 and at is not None and "wait_kv" not in at.group(0)[:-len("wait_kv(v_pos(j)")]


def test_both_query_tiles_of_plain_attention():
    text = source("attention_tc.cuh")
    assert in_order_tc(text)
    # what the check is for: either tile in the other order, or a place more, is seen
    assert not in_order_tc(text.replace("wait_p(0, j) && wait_kv(v_pos(j))", "wait_kv(v_pos(j)) && wait_p(0, j)"))
    assert not in_order_tc(text.replace("wait_p(1, j) && (j < n_a || wait_kv(v_pos(j)))", "(j < n_a || wait_kv(v_pos(j))) && wait_p(1, j)"))
    assert not in_order_tc(text + "wait_kv(v_pos(j));")


def test_both_query_tiles_of_attention_over_pages():
    text = source("attention_paged_tc.cuh")
    assert in_order_paged(text)
    assert not in_order_paged(text.replace("bool landed = false;", "bool landed = wait_kv(v_pos(j));"))
    assert not in_order_paged(text.replace("if (ok && !landed) ok = landed = wait_kv(v_pos(j)", "ok = landed = wait_kv(v_pos(j)"))


def test_no_other_ring_of_three():
    """The rings of the other kernels are of four tiles and more, which are safe in either order."""
    rings = {p.name: re.findall(r"constexpr int kRing = ([^;]+);", p.read_text()) for p in CSRC.glob("*.cuh")}
    sizes = {name: [int(x) for r in found for x in re.findall(r"(?<![=\d] )\b\d+\b", re.sub(r"D == \d+", "", r))] for name, found in rings.items() if found}
    assert {name for name, s in sizes.items() if min(s) < 4} == {"attention_tc.cuh", "attention_paged_tc.cuh"}, sizes
