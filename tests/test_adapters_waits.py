"""What the prompts' kernels do after a bounded wait that ran out, which no run on a GPU can be made to show without a
fault: read from the source."""

import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reflex_b200", "csrc", "adapters_prompt.cu")


def after(code, lines=6):
    """The lines that follow the report of a wait by its number."""
    with open(SOURCE) as f:
        text = f.read()
    assert text.count(f"atomicExch(err, {code})") >= 1
    return "\n".join(text.split(f"atomicExch(err, {code})", 1)[1].splitlines()[:lines])


def test_what_is_on_its_way_is_waited_for():
    for code, bar in ((62, "done_bar"), (63, "full_bar"), (65, "acc_full"), (67, "v_full")):
        assert re.search(r"mbar_wait\(&" + bar, after(code)), code


def test_products_before_a_wait_that_ran_out_are_committed():
    with open(SOURCE) as f:
        text = f.read()
    assert not re.search(r"if \(.*\) umma_commit\(&done_bar\)", text) and "umma_commit(&done_bar)" in text
