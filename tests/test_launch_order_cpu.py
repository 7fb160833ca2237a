"""Order of set-up steps in kernels that take tensor memory, read from their source.

A kernel that lets its dependents start (pdl_trigger) while one of its warps may still wait for tensor memory can be
locked out by them: a dependent's block takes the memory and waits for the first kernel's end.  So the allocation, then a
barrier of the block, then the trigger."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dcnv4_b200", "csrc")


def kernels():
    """(file, name, body) of every __global__ function that allocates tensor memory and launches dependents."""
    for f in sorted(os.listdir(CSRC)):
        if not f.endswith((".cu", ".cuh")):
            continue
        with open(os.path.join(CSRC, f)) as src:
            text = re.sub(r"//[^\n]*", "", src.read())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
            at = text.index("{", m.end())
            depth = 0
            for end in range(at, len(text)):
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                if depth == 0:
                    break
            body = text[at:end]
            if re.search(r"tmem_alloc\(|tcgen05\.alloc", body) and "pdl_trigger()" in body:
                yield f, m.group(1), body


FOUND = list(kernels())


def test_there_are_such_kernels():
    assert {"ns_kernel", "ns_small_kernel", "linear_kernel", "dcnv4_fwd_fused_kernel"} <= {name for _, name, _ in FOUND}


@pytest.mark.parametrize("name,body", [(n, b) for _, n, b in FOUND], ids=[n for _, n, _ in FOUND])
def test_dependents_start_behind_the_allocation(name, body):
    last = max(m.end() for m in re.finditer(r"tmem_alloc\(|tcgen05\.alloc", body))
    trigger = body.index("pdl_trigger()")
    assert last < trigger and "__syncthreads()" in body[last:trigger], name
