"""Decisions that the softmax warps of the 128-row attention kernel share, checked on the CPU.

One thread decides for a cut unit's part whether it is joined from registers and whether its CTA is the last to
arrive; the others read its word in shared memory after the four warps have met. Nothing holds the first warp back
once a meeting is complete: it may be at the CTA's second part before a warp that sleeps in its wait has read the
decision on the first. So a word that a later decision overwrites must have a meeting between its last reading and
the overwriting. This test takes the words from the kernel's source, restates the order of meetings, writes and
readings, and runs through every interleaving.
"""
import itertools
import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parent.parent / "flashlite_b200" / "csrc" / "fl_tree.cu").read_text()


def words():
    """(word of the decision on a direct join for a slot's parity, word of the last arrival) as the source names them."""
    direct = re.search(r"direct = (.+?) != 0;", SOURCE).group(1)
    last = re.search(r"if \((\*?\w+(?:\[.+?\])?) == 0\) break;", SOURCE).group(1)
    assert re.search(re.escape(direct) + r" = mbar_wait", SOURCE) and re.search(re.escape(last) + r" = mbar_wait", SOURCE)
    name = lambda text, slot: text.replace("g.slot & 1", str(slot & 1))  # noqa: E731
    return (lambda slot: name(direct, slot)), (lambda slot: name(last, slot))


def part(slot, direct, last, direct_word, last_word):
    """What each warp does at the end of one part: (write, word, value) is the first warp's alone."""
    ops = [("write", direct_word(slot), direct), ("meet",), ("read", direct_word(slot), direct)]
    if not direct:
        ops += [("meet",), ("write", last_word(slot), last), ("meet",), ("read", last_word(slot), last)]
    return ops


def wrong_readings(ops, warps=3):
    """Readings of another value than the decision's, over all interleavings (a meeting: arrive, then wait for all)."""
    wrong, seen = set(), set()
    stack = [((0,) * warps, (False,) * warps, ())]  # position, arrived at the meeting there, memory
    while stack:
        state = stack.pop()
        if state in seen:
            continue
        seen.add(state)
        at, arrived, memory = state
        for w in range(warps):
            if at[w] == len(ops):
                continue
            op, move = ops[at[w]], lambda x, v: x[:w] + (v,) + x[w + 1:]
            there, mem = at[w] + 1, dict(memory)
            if op[0] == "meet" and not arrived[w]:
                stack.append((at, move(arrived, True), memory))
                continue
            if op[0] == "meet" and any(at[o] < at[w] or (at[o] == at[w] and not arrived[o]) for o in range(warps)):
                continue  # somebody has not arrived
            if op[0] == "write" and w == 0:
                mem[op[1]] = op[2]
            if op[0] == "read" and mem.get(op[1]) != op[2]:
                wrong.add(op)
            stack.append((move(at, there), move(arrived, False), tuple(sorted(mem.items()))))
    return wrong


def test_no_decision_is_overwritten_before_it_is_read():
    """Two parts of a CTA one after the other, the second of one tile: no product makes the first warp wait."""
    direct_word, last_word = words()
    for d0, l0, d1, l1 in itertools.product((False, True), repeat=4):
        ops = part(0, d0, l0, direct_word, last_word) + part(1, d1, l1, direct_word, last_word)
        assert not wrong_readings(ops), (d0, l0, d1, l1)


def test_the_search_finds_an_overwritten_word():
    one = lambda slot: "word"  # noqa: E731
    assert wrong_readings(part(0, False, False, one, one) + part(1, True, False, one, one))
