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


# -- blocks of 256 rows: the words of nodes whose values are no numbers --------------------------------------------------------
def halves(two, bad):
    """The halves' groups and the issuing thread over items of one tile: two[i]: it has a second half, bad[i]: the first half finds such nodes in
    it. Either half has to see the item's own, no others'. A wait for o_free[1] tells a phase from the next one only, as the barrier does."""
    n = len(two)
    kinds = dict(clear=r"bad_nodes\[\(item \+ (\d)\) & 3\] = 0ull", set=r"atomicOr\(bad_here", free=r"wait_second\(\)")
    order = [[(k, int(m[1]) if k == "clear" else 0) for k, m, line in steps(t, **kinds) if "!WIDE &&" not in line]
             for t in (SOFTMAX[SOFTMAX.index("for (uint32_t item"):], RESULTS)]
    assert [k for k, _ in order[0] + order[1]].count("set") == 1 and any(k == "clear" for k, _ in order[0] + order[1])

    def first():
        program = []
        for i in range(n):
            had = sum(two[:i])

            def wait(v, had=had):
                return None if had == 0 or (v["o_free1"] - 1) % 2 == (had - 1) % 2 else False

            def part(order, i=i, wait=wait):
                out, behind_wait = [], False
                for kind, at in order:
                    if kind == "free":
                        behind_wait = True
                        continue
                    name = f"word{(i + at) % 4 if kind == 'clear' else i % 4}"

                    def step(v, kind=kind, name=name, i=i, behind_wait=behind_wait):
                        if (kind == "set" and not bad[i]) or (kind == "clear" and v[name] == ()):
                            return None
                        if behind_wait and wait(v) is False:
                            return False
                        v[name] = () if kind == "clear" else v[name] + (i,)
                    out.append(step)
                    behind_wait = False
                return out
            program += [until("s0", i + 1), *part(order[0]), add("p0"), until("pv0", i + 1), look(i), add("o_free0"), *part(order[1])]
        return program

    def look(i):
        def step(v):
            assert v[f"word{i % 4}"] == ((i,) if bad[i] else ()), "a word of another item"
        return step

    def second():
        program, k = [], 0
        for i in range(n):
            if two[i]:
                k += 1
                program += [until("s1", k), add("p1"), until("pv1", k), look(i), add("o_free1")]
        return program

    issue, k = [], 0
    for i in range(n):
        issue += [add("s0"), *([add("s1")] if two[i] else []), until("o_free0", i), until("p0", i + 1), add("pv0")]
        if two[i]:
            issue += [until("o_free1", k), until("p1", k + 1), add("pv1")]
            k += 1
    names = [f"{x}{h}" for x in ("s", "p", "pv", "o_free") for h in range(2)]
    return explore([first(), second(), issue], {**dict.fromkeys(names, 0), **{f"word{w}": () for w in range(4)}})


@pytest.mark.parametrize("two", ["2111111", "2211121", "1211112", "2222222", "2121211", "1111111", "2112112"])
def test_halves_see_the_nodes_of_their_own_item(two):
    items = [x == "2" for x in two]
    for word in range(1 << len(items)):
        halves(items, [bool(word >> i & 1) for i in range(len(items))])


def test_results_in_a_query_buffer_are_fenced_before_the_next_queries_are_copied_into_it():
    """Rows that lanes share: sums and results lie in the item's query buffer for a while. Copies write by another proxy than threads: every thread's
    writes, then its fence, a barrier of the group, then the arrival that lets the copy begin."""
    order = [k for k, _, _ in steps(RESULTS, write=r"\blanes\[tl\] = |\bat\[e \* BR\] = ", fence=r"fence_proxy_async_smem\(\)", group=r"sync_group\(\)",
                                    free=r"mbar_arrive\(&q_free")]
    last = max(i for i, k in enumerate(order) if k == "write")
    assert order.count("write") == 2 and order.count("free") == 1 and order[-1] == "free"
    fence = order.index("fence", last)
    assert "group" in order[fence:order.index("free")]
