"""How the two threads of a score row exchange their maxima in the prompt attention kernel: every order in which the
two can run, for the number of words per row that the kernel declares.

Per block a thread leaves the upper half of its maximum, meets the other at a barrier, reads the other's upper half,
meets, leaves the lower half, meets, reads the other's lower half.  Where P lies apart from the scores (heads up to 64
wide) nothing but these barriers orders a block's last read against the next block's first write; where P lies over
the scores, the next block's scores come only after both threads' P.
"""

import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-flash_b200", "csrc",
                   "prompt_attn.cu")


def thread(h, blocks, words, joined):
    """(kind, argument) steps of thread h: barriers, writes and reads of (word, thread) with the half they stand for."""
    steps = []
    for j in range(blocks):
        w = j % words
        steps += [("write", ((w, h), (j, "upper"))), ("meet", None), ("read", ((w, 1 - h), (j, "upper"))),
                  ("meet", None), ("write", ((w, h), (j, "lower"))), ("meet", None),
                  ("read", ((w, 1 - h), (j, "lower")))]
        if joined:  # the next scores wait for both threads' P
            steps.append(("meet", None))
    return steps


def wrong_reads(words, joined, blocks=4):
    """Reads that return another block's or another half's value, over every order of the two threads' steps."""
    a, b = thread(0, blocks, words, joined), thread(1, blocks, words, joined)
    seen, todo, wrong = set(), [(0, 0, ())], set()
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        i, k, memory = state
        for mine, at in ((0, i), (1, k)):
            steps = (a, b)[mine]
            if at == len(steps):
                continue
            kind, what = steps[at]
            if kind == "meet":
                if mine == 0 and k < len(b) and b[k][0] == "meet":
                    todo.append((i + 1, k + 1, memory))
                continue
            cells = dict(memory)
            if kind == "write":
                cells[what[0]] = what[1]
            elif cells.get(what[0]) != what[1]:
                wrong.add(what[1])
            todo.append((i + 1, k, tuple(sorted(cells.items()))) if mine == 0 else
                        (i, k + 1, tuple(sorted(cells.items()))))
    return wrong


@pytest.mark.parametrize("apart", [True, False])
def test_maxima_are_read_before_they_are_written_over(apart):
    m = re.search(r"TOPS = APART \? (\d) : (\d);", open(SRC).read())
    words = int(m[1 if apart else 2]) if m else 1
    assert not wrong_reads(words, joined=not apart)


def test_the_model_sees_a_missing_order():
    assert wrong_reads(1, joined=False)
