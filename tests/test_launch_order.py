"""Kernels that start while the kernel before them still runs (programmatic launch, griddepcontrol.wait) must not take what that
kernel writes through `const T* __restrict__`: the qualifier says that the memory does not change while the kernel lives, so the
compiler may read it before the wait. Read from the sources: the fault is a race, which no run shows reliably."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nibble_b200", "csrc")
# per kernel: parameters that an earlier kernel of the same chain writes
WRITTEN_BEFORE = {
    "compact_count_kernel": ["first"],
    "compact_rank_kernel": ["first", "counts"],
    "compact_move_kernel": ["new_id", "source", "n_used"],
}


def test_compact_reads_the_kernel_before_through_plain_pointers():
    with open(os.path.join(CSRC, "kv_pages.cu")) as f:
        text = f.read()
    for kernel, names in WRITTEN_BEFORE.items():
        at = re.search(r"\b" + kernel + r"\(const PageBook b, (.*?)\) \{(.*?)\n\}", text, re.S)
        assert at, kernel
        params, body = at.groups()
        assert "wait_for_previous();" in body
        for name in names:
            assert re.search(r"\*\s*" + name + r"\b", params), f"{kernel}: {name}"
            assert not re.search(r"__restrict__\s+" + name + r"\b", params), f"{kernel}: {name} is __restrict__"
            before = body.split("wait_for_previous();")[0]
            assert not re.search(r"\b" + name + r"\b", before), f"{kernel}: {name} is read before the wait"
            for use in re.finditer(r"(__ldcg\(&?)?\b" + name + r"\b( = |\[[^\]]*\] = )?", body):
                assert use.group(1) or use.group(2), f"{kernel}: {name} is read without __ldcg"
