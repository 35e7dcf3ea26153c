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


def by_one_lane(text, at, inside):
    """Whether what stands here runs in one lane of a warp alone: under such a condition, or in a function of its own that only such places call."""
    statement = text[max(text.rfind(c, 0, at) for c in ";{}") + 1:at]
    headers = [statement] + [h for _, h, a, b in inside if a <= at < b]
    if any(re.search(r"lane == 0|elect_one\(\)", h) for h in headers):
        return True
    names = [m.group(1) for h in headers for m in [re.search(r"auto (\w+) = \[&\]", h)] if m]
    calls = [m.start() for name in names for m in re.finditer(r"(?<!auto )\b%s\(" % name, text)]
    return bool(calls) and all(by_one_lane(text, c, inside) for c in calls)


@pytest.mark.parametrize("name", ["fp8_gemm.cu", "attention_tree.cu", "attention_tree_tc.cu"])
def test_a_warp_votes_on_what_it_waited_for(name):
    """Lanes that disagree on whether their wait gave up would meet in different warp-wide operations (tensor-memory loads, barriers)."""
    text = source(name)
    inside = scopes(text)
    waits = [m for m in re.finditer(r"\bmbar_wait(_at)?\(", text) if not text[:m.start()].endswith("bool ")]
    assert waits
    for m in waits:
        statement = text[max(text.rfind(c, 0, m.start()) for c in ";{}") + 1:m.start()]
        used = re.search(r"(ok|got) =|return|if \(!?$|&& $", statement)
        behind = text[text.index(";", m.start()) + 1:].lstrip()
        assert not used or behind.startswith("ok = __all_sync(0xffffffffu, ok);") or by_one_lane(text, m.start(), inside), statement + text[m.start():m.start() + 80]


def test_dependent_kernels_start_behind_the_allocation_of_tensor_memory():
    """A dependent CTA takes columns as soon as it runs and waits with them for the kernel before it. A CTA of that kernel that still had to get its own could wait for the other for ever."""
    seen = 0
    for name in sorted(f for f in os.listdir(CSRC) if f.endswith(".cu")):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for kernel in re.split(r"\b__global__\b", text)[1:]:
            allocs = [m.start() for m in re.finditer(r"\btmem_alloc\(|tcgen05\.alloc\.", kernel)]
            starts = [m.start() for m in re.finditer(r"\bpdl_launch_dependents\(\)", kernel)]
            if allocs and starts:
                seen += 1
                assert max(allocs) < min(starts), name
                # (a barrier of the block, or a wait for what has been multiplied there)
                assert re.search(r"__syncthreads\(\);|acc_full|acc_done", kernel[max(allocs):min(starts)]), name
    assert seen >= 8
