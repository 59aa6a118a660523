"""Kernels that may start before the one they depend on has ended read its results with
plain loads: the read-only path (ld.global.nc, __ldg, or a load that the compiler makes one
from a const __restrict__ pointer) is for data that nobody writes while the kernel lives."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ada-mla_b200", "csrc")


def kernels_and_files():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        starts = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
        for a, b in zip(starts, starts[1:]):
            if "griddep_wait();" in text[a:b]:
                name = re.search(r"(\w+_kernel)\s*\(", text[a:b]).group(1)
                yield os.path.basename(path), name, text[a:b], text


def test_no_read_only_loads_after_the_wait():
    seen = []
    for path, name, body, text in kernels_and_files():
        seen.append(name)
        params = body[:body.index("{")]
        assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", params), (path, name)
        assert "__ldg(" not in text and "ld.global.nc" not in text, (path, name)
    assert {"combine_kernel", "combine_rows_kernel", "merge_kernel", "tc_decode_kernel", "prefill_kernel"} <= set(seen), seen
