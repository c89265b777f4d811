"""Kernels that start before the one before them has ended (programmatic dependent launch): how the sources read what
that one writes.  Such data is not read-only for the reading kernel's lifetime, so it must not take the read-only path, which
a const __restrict__ pointer or __ldg allow: the compiler may then move the load over the wait.  A wrong order shows on no
test of results that can be relied on; the sources show it."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stk_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())          # comments out


def kernel(text, name):
    """(parameters, body) of a __global__ function."""
    at = re.search(r"\b%s\(" % name, text).end()
    close = text.index(") {", at)
    depth, end = 1, close + 3
    while depth:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
    return text[at:close], text[close + 3:end]


@pytest.mark.parametrize("file,name,pointer", [("tokens_sm100.cuh", "place_kernel", "hist"),
                                               ("int4_sm100.cuh", "int4_combine_kernel", "y")])
def test_a_pointer_to_what_the_kernel_before_writes(file, name, pointer):
    params, body = kernel(source(file), name)
    declared, = [p for p in params.split(",") if re.search(r"\b%s$" % pointer, p.strip())]
    assert "__restrict__" not in declared
    uses = [m.start() for m in re.finditer(r"\b%s\b" % pointer, body)]
    reads = [u for u in uses if not re.match(r"%s [!=]= nullptr" % pointer, body[u:])]
    assert reads and all(body[:u].endswith("load_written(") for u in reads)
    assert all(u > body.index("pdl_wait()") for u in reads)


def test_the_second_4_bit_product_reads_its_inputs_so():
    text = source("int4_sm100.cuh")
    assert "__ldg" not in text
    load = text[text.index("void load(const Int4Args"):]
    assert "load_written(" in load[:load.index("\n  }\n")]
    # ... and behind the wait: the loads are those of an item or of what is made of an entry's inputs before its items
    _, body = kernel(text, "int4_matvec_kernel")
    wait = body.rindex("pdl_wait()")
    assert all(m.start() > wait for m in re.finditer(r"int4_(item|sums)<", body))


def test_a_block_that_gives_up_a_wait_waits_for_its_copies():
    """A bulk copy that lands after its block has ended would write into another block's shared memory.  (No test makes a
    copy late: the sources show the wait, after the items, for what each warp has started.)"""
    text = source("int4_sm100.cuh")
    _, body = kernel(text, "int4_matvec_kernel")
    end = body[body.rindex("while (item.next("):]
    assert re.search(r"if \(\*static_cast<volatile int\*>\(&sm\.stuck\) != 0\) int4_drain\([^;]*cursor\.head\);", end)
    drain = text[text.index("void int4_drain("):]
    assert "mbar_wait(" in drain[:drain.index("\n}\n")]
