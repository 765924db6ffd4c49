"""CPU model of the barriers between the issuing warp, the tensor core and the
softmax warps of kv4_attn_tc_kernel: every order in which they can run is
walked, with the softmax's waits taken from the kernel's source.

An mbarrier wait names a parity, not a phase: it passes when the newest
completed phase has that parity, and on a fresh barrier for parity 1. So a wait
is right only while the barrier is at most one phase short of the one meant.
The model's barriers count completed phases and answer waits that way; each wait
passed is then held against what it is there for."""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "servoflow_b200", "csrc",
                   "kv4_attn_tc.cu")


def source_waits():
    """(barrier, parity expression) of the softmax's wait for Sᵀ, before it rescales Oᵀ, and for the end."""
    with open(SRC) as f:
        body = f.read().split("── softmax: thread = key", 1)[1]
    grab = lambda pattern: re.search(pattern, body).groups()
    return {"s": grab(r"wait\((bar_s\(u\)), ([^;]+)\);"),
            "rescale": grab(r"wait\((kBarO), ([^;]+)\);"),
            "end": grab(r"if \(ntl (?:>= 1|> 0)\) wait\((\w+), ([^;]+)\);")}


def parity(expr, **names):
    return eval(expr.replace("/", "//"), {}, names)


def walk(ntl, rescale, waits):
    """All reachable states of one softmax warp (the barrier of the others' arrivals
    is open as soon as this one has arrived: the least that can hold it back), the
    issuing warp and the tensor core. Returns what a wait let through too early."""
    # issuing warp: Sᵀ of two tiles, then P·V of a tile before Sᵀ of the tile two later
    program = [("s", j) for j in range(min(2, ntl))]
    for j in range(ntl):
        program += [("wait_p", j), ("o", j)] + ([("s", j + 2)] if j + 2 < ntl else [])
    program.append(("end", 0))
    commits = {"s": lambda j: (f"s{j & 1}",), "o": lambda j: ("kBarO",), "end": lambda j: ("kBarDone",)}

    def bar_of(name, j):
        return f"s{j & 1}" if name.startswith("bar_s") else name

    def passes(done, bar, par):
        return (done.count(bar) & 1) != par

    found = set()
    # state: issuing warp's step, MMAs issued, MMAs completed, softmax tile and step
    todo, seen = [(0, (), 0, 0, 0)], set()
    while todo:
        st = todo.pop()
        if st in seen:
            continue
        seen.add(st)
        pc, issued, ndone, tile, step = st
        done = tuple(b for op in issued[:ndone] for b in commits[op[0]](op[1]))
        pv_done = sum(op[0] == "o" for op in issued[:ndone])
        s_done = sum(op[0] == "s" for op in issued[:ndone])
        if ndone < len(issued):                            # the tensor core, in order
            todo.append((pc, issued, ndone + 1, tile, step))
        if pc < len(program):                              # the issuing warp
            op = program[pc]
            if op[0] != "wait_p":
                todo.append((pc + 1, issued + (op,), ndone, tile, step))
            elif tile > op[1]:                             # the softmax has arrived for this tile
                todo.append((pc + 1, issued, ndone, tile, step))
        if tile < ntl:                                     # the softmax
            if step == 0:
                bar, expr = waits["s"]
                if passes(done, bar_of(bar, tile), parity(expr, j=tile)):
                    if s_done <= tile or pv_done < tile - 1:
                        found.add("s")                     # its logits, and its buffer of P
                    todo.append((pc, issued, ndone, tile, 1))
            elif rescale and tile > 0:
                bar, expr = waits["rescale"]
                if passes(done, bar, parity(expr, j=tile)):
                    if pv_done < tile:
                        found.add("rescale")
                    todo.append((pc, issued, ndone, tile + 1, 0))
            else:
                todo.append((pc, issued, ndone, tile + 1, 0))
        elif step == 0:
            bar, expr = waits["end"]
            if passes(done, bar, parity(expr, ntl=ntl)):
                if pv_done < ntl:
                    found.add("end")
                todo.append((pc, issued, ndone, tile, 1))
    assert any(st[0] == len(program) and st[3:] == (ntl, 1) for st in seen)      # the walk gets to the end
    return found


@pytest.mark.parametrize("rescale", [False, True])
@pytest.mark.parametrize("ntl", [1, 2, 3, 4, 5, 6, 7])
def test_no_wait_is_answered_by_another_phase(ntl, rescale):
    assert walk(ntl, rescale, source_waits()) == set()


def test_the_model_finds_a_wait_that_is_two_phases_short():
    waits = dict(source_waits(), end=("kBarO", "(ntl - 1) & 1"))
    assert walk(1, False, waits) == set()                  # one tile: its only phase
    for ntl in (2, 3, 4, 5):
        assert walk(ntl, False, waits) == {"end"}


def test_the_end_is_committed_behind_the_last_product():
    """kBarDone is committed once, after the loop that issues every tile's product,
    and not where that loop was left early."""
    with open(SRC) as f:
        src = f.read()
    assert len(re.findall(r"mma_commit\(&bars\[kBarDone\]\)", src)) == 1
    tail = src.split("for (int j = 0; j < ntl && ok; ++j) {", 1)[1]
    assert re.search(r"if \(ok\) mma_commit\(&bars\[kBarDone\]\);", tail)
