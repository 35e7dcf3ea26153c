"""How the kernels of the 8-bit operators leave when a bounded wait gives up, read from their sources: a wait that runs out cannot be had on a GPU without breaking a kernel."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "et_b200", "csrc")


def source(name):
    """A source without its comments and its inline assembly's texts."""
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r'"(?:\\.|[^"\\])*"', '""', re.sub(r"//[^\n]*", "", text))


def scopes(text):
    """(where its header starts, header, where its body starts, where it ends) of every pair of braces."""
    found, stack, last = [], [], 0
    for m in re.finditer(r"[{};]", text):
        if m.group() == "{":
            stack.append((last, text[last:m.start()], m.end()))
        elif m.group() == "}" and stack:
            found.append((*stack.pop(), m.start()))
        # (a for's own semicolons do not end its header)
        if m.group() != ";" or text.count("(", last, m.start()) == text.count(")", last, m.start()):
            last = m.end()
    return found


def test_no_warp_leaves_a_loop_whose_barriers_count_it():
    """bar.sync counts the threads of all warps that share it. A warp that left at its limit would leave the others waiting for it without one."""
    text = source("fp8_gemm.cu")
    loops = [(a, b) for _, header, a, b in scopes(text) if re.search(r"\bfor \(", header) and "few_barrier();" in text[a:b]]
    assert len(loops) == 1
    body = text[slice(*loops[0])]
    assert body.count("few_barrier();") == 2 and "acc_full" in body
    assert not re.search(r"\b(break|return|goto)\b", body)
