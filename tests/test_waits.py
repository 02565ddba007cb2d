"""What the kernels do when a bounded wait has run out, by their source: no test makes one run out, since that would take a GPU that hangs."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quant_cast_bench_b200", "csrc")


def source(name):
    """The text of a file of csrc/ without comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", ["int8.cu", "kv_prompt.cu"])
def test_copies_settle_after_the_last_barrier(name):
    """A CTA in which a wait ran out waits for its copies once no thread issues any more, and before it gives up its memory."""
    text = source(name)
    assert len(re.findall(r"\bsettle\(", text)) == 1
    at = text.index("settle(")
    assert text[:at].rstrip().endswith("__syncthreads();") and "tmem_free(" in text[at:at + 200]


def loops_that_arm(text):
    """The bodies of the innermost loops that arm a transaction barrier."""
    for m in re.finditer(r"\bmbar_expect_at\(", text):
        start = text.rindex("for (", 0, m.start())
        yield text[start:m.end()]


@pytest.mark.parametrize("name", ["int8.cu", "kv_prompt.cu"])
def test_no_barrier_is_armed_behind_a_wait_that_ran_out(name):
    loops = list(loops_that_arm(source(name)))
    assert loops
    for body in loops:
        assert "mbar_reached(" in body and "mbar_wait_at(" not in body and "break;" in body
