"""The kernels of 4-bit floating point and of the balance loss are launched before the kernel ahead of them has ended, some through a
lambda or with their own launch attributes: each waits for it, touches nothing but its own shared memory and the L2 before, and reads what
others wrote with loads that the compiler may not move over the wait."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "suzuku-engine-q4_b200", "csrc")
FILES = ("q4b_fp4.cu", "q4b_fp4_tc.cu", "q4b_balance.cu")


def _text(name):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(CSRC, name)).read(), flags=re.S)


def _kernels():
    for name in FILES:
        for part in re.split(r"(?<=\n)}\n", _text(name)):
            if "__global__" in part:
                body = part[part.rindex("__global__"):]
                yield re.search(r"\b(\w+_k)\(", body).group(1), body


KERNELS = dict(_kernels())


def test_all_kernels_of_the_files_are_seen():
    launched = set()
    for name in FILES:
        launched |= set(re.findall(r"\b(?:go|q4b_launch|cudaLaunchKernelEx)\((?:&cfg, )?(\w+_k)\b", _text(name)))
    assert launched == set(KERNELS) == {"quantize_k", "values_k", "put_k", "few_k", "tc_k", "rows_k"}


@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_waits_before_it_reads_or_writes(kernel):
    body = KERNELS[kernel]
    assert body.count("q4b_pdl_wait();") == 1
    head = body[body.index("{"):body.index("q4b_pdl_wait();")]
    # parameters and their sizes may be read, not what they point to
    assert not re.search(r"\b(?:a\.\w+|codes|scales|out|w)\s*\[", head), head
    assert not re.search(r"\*\s*a\.|\batomic|\bload8|\b__ld|ld\.global|st\.global|bulk_load|tma_load|\bwait\(", head)
    for to in re.findall(r"\*reinterpret_cast<[^>]*>\(([^+)]*)", head):
        assert to.strip() in ("ring", "smem_raw")                         # (shared memory)
    for op in re.findall(r'asm volatile\(\s*"([\w.:]+)', head):
        assert op.startswith("fence.") or ".prefetch." in op, op
    # a lambda that is made ahead of the wait is called behind it
    for name in re.findall(r"auto (\w+) = \[&\]", head):
        assert not re.search(r"[^.\w]%s\(" % name, head[head.index("auto " + name) + len(name) + 8:])


@pytest.mark.parametrize("name", FILES)
def test_reads_plainly(name):
    text = _text(name)
    assert "__restrict__" not in text and "ld.global.nc" not in text
    loads = re.findall(r"\b__ld(?:g|cg|cs|ca|lu|cv)\(([\w.]+)", text)
    # the clusters' sums, which this launch's CTAs wrote: read behind the counter that the last of them takes, and a fence
    assert loads == (["a.part"] if name == "q4b_balance.cu" else [])
    if loads:
        body = KERNELS["rows_k"]
        counter, fence, load = body.index("atomicInc(a.done"), body.rindex("__threadfence();"), body.index("__ldcg(a.part")
        assert body.index("q4b_pdl_wait();") < body.index("__threadfence();") < counter < fence < load
