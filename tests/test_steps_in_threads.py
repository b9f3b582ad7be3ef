"""Two engines in two threads at once, as the C interface's handles allow: what a step sets for its own operators is the
thread's."""

import threading

import pytest
import torch

from reflex_b200 import ops


def beside(enter, read):
    """What each of two threads reads while both are inside blocks of their own, the other's the later one."""
    inside, both, done, seen = threading.Event(), threading.Event(), threading.Event(), {}

    def other():
        inside.wait(10)
        with enter("other"):
            seen["other"] = read()
            both.set()
            done.wait(10)

    t = threading.Thread(target=other)
    t.start()
    with enter("mine"):
        inside.set()
        assert both.wait(10)
        seen["mine"] = read()
        done.set()
        t.join()
    assert read() is None
    return seen


def test_each_steps_adapters():
    got = beside(lambda who: ops.use_adapters(who), ops.active_adapters)
    assert got == {"mine": "mine", "other": "other"}


def test_a_thread_begins_without_adapters():
    seen = []
    with ops.use_adapters("mine"):
        t = threading.Thread(target=lambda: seen.append(ops.active_adapters()))
        t.start()
        t.join()
    assert seen == [None]


def test_each_steps_working_memory():
    from reflex_b200.ops import workspace

    spaces = {who: workspace.Workspace("cpu") for who in ("mine", "other")}
    got = beside(lambda who: workspace.use(spaces[who]), workspace.active)
    assert got == spaces
