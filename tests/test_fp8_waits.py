"""The 8-bit kernels that may start before the one before them has ended, by reading their source: nothing that an earlier kernel
wrote is loaded as read-only data, and pointers to it are taken behind the wait."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yamoe_b200", "csrc")
#: file: kernels that start early, and how often the file launches such a kernel
EARLY = {"fp8_quant.cuh": (["quantize_rows_kernel", "quantize_tile_kernel"], 2), "fp8_gemm.cuh": (["fp8_gemm_kernel"], 1)}


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_early_kernels_are_known():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cuh", ".cu")) and name != "common.cuh":
            text = source(name)
            launches = text.count("launch_early(") + text.count("cudaLaunchAttributeProgrammaticStreamSerialization")
            assert launches == EARLY.get(name, ([], 0))[1], name


@pytest.mark.parametrize("name,kern", [(f, k) for f in sorted(EARLY) for k in EARLY[f][0]])
def test_early_kernels_read_behind_the_wait(name, kern):
    text = source(name)
    start = text.index("\n%s(" % kern)
    body = text[start:text.index("\n}\n", start)]
    wait = body.index("pdl_wait()")
    assert all(m.start() > wait for m in re.finditer(r"after_wait\(", body))
    assert "__ldg(" not in body and "__restrict__" not in body
    for load in ("tma_load_3d(", "copy_float(", "pad_off["):
        assert all(m.start() > wait for m in re.finditer(re.escape(load), body)), load


@pytest.mark.parametrize("name", sorted(EARLY))
def test_no_read_only_loads(name):
    assert "__ldg(" not in source(name)
