"""What the tensor cores' attention with a window does where one of its bounded
waits runs out, by reading: a model of the warps that meet at barriers, which
leaves as the kernel's source says, and the copies that a block has under way.
No GPU: there the waits do not run out."""
import itertools
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).parent.parent / "neuralscript_b200" / "csrc" / "attention_window_tc.cu").read_text()


def between(start, end):
    return SOURCE[SOURCE.index(start):].split(end, 1)[0]


def leaves(kernel):
    """Whether a warp whose wait ran out meets the others: always, or while a meeting of all is still to come."""
    rule = re.search(r"auto await = .*?\n\s+if \((!ok(?: && !last)?)\) meet<", between(f"{kernel}(", "// -----"), re.S)
    return {"!ok": "always", "!ok && !last": "before the last"}[rule[1]]


def stuck(program, ran_out, rule):
    """Two warps through `program` (w: a wait, m: a meeting), each with the waits that run out for it: whether one stands
    at a meeting that the other has passed by."""
    def warp(out):
        waits = 0
        for i, op in enumerate(program):
            if op == "m":
                if (yield False):
                    return
            else:
                if waits in out:
                    if rule == "always" or "m" in program[i:]:
                        yield True
                    return
                waits += 1

    warps = [warp(out) for out in ran_out]
    gone = [next(w, None) for w in warps]
    while any(g is not None for g in gone):
        if any(g is None for g in gone):
            return True
        some = any(gone)
        for i, w in enumerate(warps):
            try:
                gone[i] = w.send(some)
            except StopIteration:
                gone[i] = None
    return False


# D's sum; with the pass before, its waits, all have read, and the second sum; the tiles' waits and the last product's
QUERIES = ["m" + "wwwww", "m" + "ww" + "mm" + "wwwww"]
# tile by tile: scores, maxima, products where a maximum rises; the last product, sums
FORWARD = ["wm" + "wwm" + "wm" + "wwm" + "wm"]


@pytest.mark.parametrize("kernel,program", [("window_tc_bwd_q_kernel", p) for p in QUERIES] + [("window_tc_fwd_kernel", p) for p in FORWARD])
def test_nobody_stands_at_a_barrier_that_another_will_not_reach(kernel, program):
    rule, n = leaves(kernel), program.count("w")
    for ran_out in itertools.product([set()] + [{i} for i in range(n)], repeat=2):
        assert not stuck(program, ran_out, rule), ran_out


def test_the_model_finds_who_stands():
    assert stuck("mw", ({0}, set()), "always") and not stuck("mw", ({0}, set()), "before the last")
    assert not stuck("wm", ({0}, set()), "always") and not stuck("wm", ({0}, {0}), "before the last")


def test_a_given_up_copy_is_awaited():
    """A loader that gives up a copy with rows to clear waits for it all the same."""
    body = between("bool fill_slot(", "\n}\n")
    given_up = re.search(r"if \(!wait\(landed, tails(?:\+\+)?\)\)(.*?)return false;", body, re.S)[1]
    assert "ptx::mbar_wait(landed, tails & 1, nullptr, 0)" in given_up
