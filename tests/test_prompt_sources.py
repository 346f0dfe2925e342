"""CPU-only: an order in the prompt kernels' source that no run shows, since what goes wrong without it is a wait without a limit."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hqekv_b200", "csrc")


def kernels():
    """(name, body) of every kernel, without comments."""
    found = []
    for name in sorted(f for f in os.listdir(CSRC) if f.endswith(".cu")):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
        text = re.sub(r"__launch_bounds__\([^()]*\)", "", text)
        for m in re.finditer(r"__global__\s+void\s+(\w+)\s*\([^{;]*\)\s*\{", text):
            end = text.index("\n}", m.end())
            found.append((m.group(1), text[m.end():end]))
    return found


WITH_TENSOR_MEMORY = [(n, b) for n, b in kernels() if "tmem_alloc(" in b]


def test_both_kernels_are_looked_at():
    assert {n for n, _ in WITH_TENSOR_MEMORY} == {"prompt_kernel", "importance_kernel"}


@pytest.mark.parametrize("name, body", WITH_TENSOR_MEMORY, ids=[n for n, _ in WITH_TENSOR_MEMORY])
def test_tensor_memory_before_the_next_kernel(name, body):
    """A CTA lets the next kernel start only when it has its tensor memory: a CTA of that kernel which shared the SM could take all
    of it and would keep it while it waits for this kernel's end."""
    alloc = body.index("tmem_alloc(")
    got = body.index("__syncthreads()", alloc)
    announce = [m.start() for m in re.finditer(r"launch_dependents", body)]
    assert len(announce) == 1 and alloc < got < announce[0] < body.index("griddepcontrol.wait")


def branches(body):
    """What each role of a kernel's warps does."""
    parts = re.split(r"\n  (?:\} else )?if \(warp [^\n]*\) \{\n", body)
    return parts[1:]


def test_warps_that_elect_give_up_as_one():
    """An elected thread needs its whole warp: a warp whose lanes left a wait that ran out one by one would wait for them for good.  The
    waits of one thread belong where that thread alone is at work."""
    found = 0
    for name, body in WITH_TENSOR_MEMORY:
        for part in branches(body):
            if "elect_one()" in part:
                found += 1
                assert "bar_wait_one(" not in part and "bar_wait(" in part, name
        for m in re.finditer(r"bar_wait_one\(", body):
            assert "lane == 0" in body[max(0, m.start() - 1200):m.start()], name
    with open(os.path.join(CSRC, "tensor.cuh")) as f:
        assert re.search(r"bool bar_wait\([^)]*\) \{\s*return __all_sync\(0xffffffffu, bar_wait_one\(", f.read())
    assert found >= 2


def test_work_in_flight_is_waited_for_whichever_role_gave_up():
    """A role ends with its own waits in order where another one has given up, too.  So what is under way (products that read shared memory
    and write tensor memory, copies into shared memory) is waited for when all roles have ended, if any of them gave up."""
    for name, body in WITH_TENSOR_MEMORY:
        ended = body.rindex("__syncthreads()", 0, body.rindex("__syncthreads()"))
        last = re.match(r"__syncthreads\(\);\s*fence_after\(\);\s*if \(\*stop\) \{(.*?)\n    __syncthreads\(\);\n  \}\s*if \(warp == 8\) tmem_free", body[ended:], re.S)
        assert last, name
        for what in ("sh.drained", "sh.full[" if name == "importance_kernel" else "sh.kv_full["):
            assert what in last.group(1), (name, what)
        assert not re.search(r"(?<!next_full\), )bar_drain\((?!smem_u32\(&sh\.next_full)", body[:ended]), name
