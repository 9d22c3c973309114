"""The gather of `experts_fp8` reads the token rows before it waits for the routing kernel in front of it.  That is right as long as
that kernel is launched plainly, so that it begins behind all that wrote them.  By reading the sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yamoe_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def body(text, head):
    start = text.index(head)
    return text[start:text.index("\n}\n", start)]


def test_only_the_rows_are_read_before_the_wait_and_only_in_the_gather():
    text = body(source("fp8_quant.cuh"), "\nquantize_rows_kernel(")
    plain, gather = "if (d.flat_row == nullptr) pdl_wait();", "if (d.flat_row != nullptr) pdl_wait();"
    assert text.count("pdl_wait()") == 2 and text.count(plain) == text.count(gather) == 1
    before, between, behind = text[:text.index(plain)], text[text.index(plain) + len(plain):text.index(gather)], \
        text[text.index(gather) + len(gather):]
    # nothing is touched before the first wait; between the two, x alone is loaded and nothing stored
    assert "after_wait(" not in before and ".load<" not in before and "d.q" not in before and "d.scale" not in before
    assert re.findall(r"after_wait\(([^)]*)\)", between) == ["x"] and between.count("load<VEC>(src") == 1
    for word in ("d.q", "d.scale", "flat_row[", "flat_row)"):
        assert word not in between, word
    assert "after_wait(d.flat_row)" in behind and "after_wait(x)" not in behind


def test_the_gather_comes_right_behind_the_routing():
    text = source("yamoe_b200.cu")
    calls = re.findall(r"\b(launch_route_rows|fp8_gather|fp8_gate_up|fp8_down|launch_combine)<", body(text, "static int experts_fp8_impl("))
    assert calls == ["launch_route_rows", "fp8_gather", "fp8_gate_up", "fp8_down", "launch_combine"]
    # nobody else gathers, and nobody else gives the kernel a table
    gathers = [n for n in sorted(os.listdir(CSRC)) for _ in re.findall(r"\bfp8_gather<\w+>\(", source(n)) if n.endswith((".cu", ".cuh"))]
    assert set(gathers) <= {"yamoe_b200.cu", "fp8.cu"} and gathers.count("yamoe_b200.cu") == 1
    assert len(re.findall(r"launch_quantize_rows<", source("fp8.cu"))) == 2
    assert body(source("fp8.cu"), "static int quantize_impl(").count("nullptr, 0};") == 1


def test_routing_kernels_are_launched_plainly():
    text = source("routing.cuh")
    launched = set(re.findall(r"(\w+)(?:<T>)?<<<", text))
    assert {"kern", "route_count_kernel", "route_place_kernel"} <= launched and "auto kern = route_cluster_kernel<T>;" in text
    for word in ("launch_pdl_opt", "launch_early", "cudaLaunchKernelEx", "ProgrammaticStreamSerialization", "pdl_wait"):
        assert word not in text, word
