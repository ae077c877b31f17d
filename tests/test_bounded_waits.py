"""CPU: what follows a bounded wait that ran out ends too.

Every wait of the tensor-core kernels has a limit, behind which the kernel records an error and returns. That holds only if nobody is left
at an unbounded barrier: two warps that meet at one must leave together, and so must the lanes of a warp that goes on to
collectives. The first test runs every outcome of the waits of the two epilogue warps that share 32 rows of a tile (sm100_lora.cu); the
others read from the sources that the kernels have the form that passes."""
import itertools
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kernel_set_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _warp(waits, chunks, together):
    """One epilogue warp: a wait before the loop and one per chunk, each of which may run out; yields its word at each barrier."""
    ok = waits[0]
    if together:
        ok = yield ok
    if not ok:
        return
    for j in range(chunks):
        ok = waits[1 + j]
        if not together and not ok:
            return
        ok = yield ok
        if not ok:
            return


def _stuck(a, b):
    """Runs two warps that meet at one barrier; whether one is left waiting at it."""
    def step(w, answer):
        try:
            return True, w.send(answer)
        except StopIteration:
            return False, None
    answer = None
    while True:
        (at_a, ok_a), (at_b, ok_b) = step(a, answer), step(b, answer)
        if at_a != at_b:
            return True
        if not at_a:
            return False
        answer = ok_a and ok_b


@pytest.mark.parametrize("chunks", [0, 1, 2, 3])
def test_pairs_leave_together(chunks):
    outcomes = list(itertools.product([True, False], repeat=1 + chunks))
    pairs = list(itertools.product(outcomes, outcomes))
    assert not any(_stuck(_warp(x, chunks, True), _warp(y, chunks, True)) for x, y in pairs)
    # what the model finds where each leaves for itself
    assert any(_stuck(_warp(x, chunks, False), _warp(y, chunks, False)) for x, y in pairs) == (chunks > 0)


def test_named_barriers_behind_bounded_waits_are_votes():
    text = _source("sm100_lora.cu")
    assert not re.search(r"\bbar(?:rier)?(?:\.cta)?\.sync\b", text), "a named barrier that a warp may be left at"
    assert text.count("bar.red.and.pred") == 1
    assert len(re.findall(r"=\s*pair_agrees\(", text)) == 2      # before the loop over the chunks, and in it


def test_warps_leave_waits_as_one():
    """Result of every wait that a whole warp takes: by vote. Not so the producers' (each thread for itself, no collective behind)
    and the waits for copies on the way out, whose result nobody uses."""
    alone = {"0x31", "0x42", "0x45", "0x52"}
    found = 0
    for name in ("sm100_lora.cu", "moe_backward.cu"):
        for m in re.finditer(r"(all_lanes\((?:sm100::)?)?\bmbar_wait(?:_long|_cluster)?\(wctx[^;]*?(0x[0-9a-f]+)\)", _source(name)):
            found += 1
            assert m[1] or m[2] in alone, (name, m[0])
    assert found >= 15
