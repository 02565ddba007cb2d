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


def test_few_queries_a_lane_whose_wait_ran_out_stops_copying():
    """kv_attention.cu arms and copies in fetch(), both only in lanes whose waits were met; and a CTA settles behind its last unit."""
    text = source("kv_attention.cu")
    assert "mbar_wait" not in text
    fetch = text[text.index("const auto fetch"):text.index("seek();", text.index("const auto fetch"))]
    assert "on_time = !(f_stage & SP_LATE)" in fetch
    assert re.findall(r"if \(([^\n]*)\) mbar_expect_at\(", text) == ["lane == 0 && on_time"]
    assert re.findall(r"if \(([^\n]*)\) bulk_load_at\(", text) == ["ok"] and "num_pages && on_time;" in fetch
    waits = re.findall(r"if \(!copied\(.*?\n            \}", text, re.S)
    assert len(waits) == len(re.findall(r"\bcopied\(", text)) - 1 == 1 and "f_stage |= SP_LATE;" in waits[0] and "out_of_time = 1;" in waits[0]
    end = text.index("settle(smem")
    assert text.rindex("named_barrier(", 0, end) > text.rindex("fetch()", 0, end)


@pytest.mark.parametrize("name", ["int8.cu", "kv_attention.cu", "kv_prompt.cu"])
def test_copies_are_ordered_behind_the_overlapped_predecessor(name):
    """Between the wait for the predecessor's end and the first copy by the async proxy stands a fence between the proxies."""
    text = source(name)
    fences = [m.start() for m in re.finditer(r"\bpdl_copies_fence\(\)", text)]
    kernel = text.index("__grid_constant__ CUtensorMap map_w") if name == "int8.cu" else text.index("kv_attn_split_kernel(" if name == "kv_attention.cu" else "kv_prompt_kernel(const")
    wait = text.index("pdl_wait()", kernel)
    issue = text.index({"int8.cu": "tma_load_2d_at(", "kv_prompt.cu": "bulk_load_at(", "kv_attention.cu": "fetch();"}[name], kernel)
    assert len(fences) == 1 and wait < fences[0] < issue
