"""How the threads of a block leave the attention cache's kernel for many columns when a wait runs out, restated on the CPU.

Each kind of warp loops over the steps: it works (a wait may run out there, which it records), meets the others at
the block's barrier, and asks whether to leave. Between the barrier and the question a thread ahead may already
record a failure of the next step. Every order of two threads is tried.
"""
from __future__ import annotations

import pytest


def orders_end(leaves, record, steps, fails):
    """Whether every interleaving of two threads ends with both out after the same number of barriers. `fails`: (thread,
    step) whose wait runs out."""
    # a thread is (step, place): 0 works, 1 at the barrier, 2 asks, 3 out
    start = ((0, 0), (0, 0), 0)
    seen, todo, good = {start}, [start], True
    while todo:
        a, b, flag = todo.pop()
        nexts = []
        if a[1] == b[1] == 1:
            nexts.append(((a[0], 2), (b[0], 2), flag))
        for t, me in enumerate((a, b)):
            if me[1] == 0:
                f = record(me[0]) if (t, me[0]) in fails else flag
                new = (me[0], 1)
            elif me[1] == 2:
                f = flag
                new = (me[0], 3) if leaves(flag, me[0]) or me[0] + 1 == steps else (me[0] + 1, 0)
            else:
                continue
            nexts.append((new, b, f) if t == 0 else (a, new, f))
        if not nexts:
            good &= a[1] == b[1] == 3 and a[0] == b[0]
        for n in nexts:
            if n not in seen:
                seen.add(n)
                todo.append(n)
    return good


@pytest.mark.parametrize("fails", [set(), {(0, 0)}, {(1, 1)}, {(0, 1), (1, 1)}, {(0, 3)}, {(1, 2), (0, 3)}])
def test_every_thread_leaves_after_the_same_step(fails):
    assert orders_end(lambda flag, i: flag != 0 and flag <= i + 1, lambda i: i + 1, 4, fails)


def test_a_plain_flag_would_leave_a_thread_at_the_barrier():
    assert orders_end(lambda flag, i: flag != 0, lambda i: 1, 4, {(0, 0)})
    assert not orders_end(lambda flag, i: flag != 0, lambda i: 1, 4, {(0, 1)})
