"""Orders that the attention of drafted nodes rests on, in every interleaving of its threads (CPU). The steps are read from the kernel's source in their
order; what lies in shared memory is followed through all states that the waits allow."""
import os
import re

import pytest

from gllm_b200 import build

SOURCE = open(os.path.join(build.CSRC, "draft", "draft_attention.cu")).read()
SOFTMAX = SOURCE[SOURCE.index("---- softmax"):SOURCE.index("---- results;")]
RESULTS = SOURCE[SOURCE.index("---- results;"):SOURCE.index("Joins the parts of the unit")]


def steps(text, **kinds):
    """[(kind, match, the code line it stands in)] in the order of the source, without comments."""
    lines = [re.sub(r"//.*", "", x) for x in text.split("\n")]
    return [(kind, m, line) for line in lines for _, kind, m in
            sorted(((m.start(), kind, m) for kind, p in kinds.items() for m in re.finditer(p, line)), key=lambda x: x[0])]


def explore(programs, start):
    """All states of `programs`: lists of steps, each a function of the variables (a dict) that changes them, or returns False where it has to
    wait. Fails where nobody can go on before all have ended."""
    freeze = lambda pcs, v: (pcs, tuple(sorted(v.items())))
    first = freeze((0,) * len(programs), start)
    todo, known = [first], {first}
    while todo:
        pcs, held = todo.pop()
        moved = False
        for a, program in enumerate(programs):
            if pcs[a] == len(program):
                continue
            v = dict(held)
            if program[pcs[a]](v) is False:
                continue
            moved = True
            new = freeze(pcs[:a] + (pcs[a] + 1,) + pcs[a + 1:], v)
            if new not in known:
                known.add(new)
                todo.append(new)
        assert moved or all(pc == len(p) for pc, p in zip(pcs, programs)), f"nobody goes on: {pcs}"
    return len(known)


def add(name, by=1):
    def step(v):
        v[name] += by
    return step


def until(name, least):
    return lambda v: None if v[name] >= least else False


# -- the maximum of a row that two warps have between them ------------------------------------------------------------------
def pair(wide, tiles=4):
    """The two warps of a row and the issuing thread. After tile k both have to see the maximum of tiles 0 .. k of both, no more."""
    order = steps(SOFTMAX, meet=r"\bsync_pair\(\);", max=r"atomicMax\(&row_max", look=r"volatile int\*>\(&row_max", hand=r"mbar_arrive\(&p_full")
    assert sorted({k for k, _, _ in order}) == ["hand", "look", "max", "meet"]

    def warp(me):
        program, met = [], 0
        for k in range(tiles):
            program.append(until("scores", k + 1))
            for kind, _, line in order:
                if kind == "meet" and ("!WIDE" in line and wide or "t > it.t0" in line and k == 0):
                    continue
                if kind == "meet":
                    met += 1
                    program += [add(f"met{me}"), until(f"met{1 - me}", met)]
                elif kind == "max":
                    program.append(lambda v, x=2 * k + me + 1: v.update(row_max=max(v["row_max"], x)))
                elif kind == "hand":
                    program.append(add("probabilities"))
                else:
                    def look(v, k=k):
                        assert v["row_max"] == 2 * k + 2, "the maximum of a tile to come"
                    program.append(look)
        return program

    issue = [add("scores")]
    for k in range(tiles):
        wait = until("probabilities", 2 * (k + 1))
        issue += [wait, add("scores")] if wide else [add("scores"), wait]
    return explore([warp(0), warp(1), issue], dict(scores=0, probabilities=0, met0=0, met1=0, row_max=0))


@pytest.mark.parametrize("wide", [True, False])
def test_both_warps_of_a_row_see_one_maximum(wide):
    # the issuing thread's orders: S of the next tile behind its wait for P of this one (blocks of 256 rows), or before it
    two_halves = SOURCE[SOURCE.index("if constexpr (WIDE) {"):SOURCE.index("// S of tile `tile_no`")]
    assert two_halves.index("wait(&p_full[h]") < two_halves.index("if (more) issue_s(")
    narrow = SOURCE[SOURCE.index("// S of tile `tile_no`"):SOURCE.index("umma_commit(mma_end)")]
    assert narrow.index("scores(g + 1") < narrow.index("wait<true>(&p_full[")
    assert pair(wide) > 10
