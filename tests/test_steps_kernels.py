"""Kernels of the expert layer's steps, by reading their source: what starts early reads nothing before it has waited, waits of whole warps have
one outcome, tables and shared memory hold what the kernels put there."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yamoe_b200", "csrc")
#: file: its kernels
KERNELS = {"token_sort.cuh": ["sort_small_kernel", "sort_count_kernel", "sort_rank_kernel", "sort_copy_kernel", "combine_tokens_kernel",
                              "link_rows_kernel", "combine_backward_kernel"],
           "glu.cuh": ["glu_forward_kernel", "glu_backward_kernel"],
           "int8_quant.cuh": ["int8_rows_quantize_kernel", "int8_columns_quantize_kernel"],
           "int8_gemm.cuh": ["int8_pair_kernel", "int8_rows_kernel"]}


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def kernel(text, name):
    start = text.index("\n%s(" % name)
    return text[start:text.index("\n}\n", start)]


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_kernels_are_known(name):
    text = source(name)
    assert re.findall(r"\n(\w+_kernel)\(", text) == KERNELS[name]
    assert "<<<" not in text                   # all by launch_behind and launch_clusters


def test_nobody_else_starts_kernels_that_way():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cuh", ".cu")) and name not in KERNELS and name != "common.cuh":
            assert "launch_behind(" not in source(name) and "launch_clusters(" not in source(name), name


@pytest.mark.parametrize("name,kern", [(f, k) for f in sorted(KERNELS) for k in KERNELS[f]])
def test_nothing_is_read_or_written_before_the_wait(name, kern):
    body = kernel(source(name), kern)
    assert body.count("pdl_wait()") == body.count("pdl_trigger()") == 1
    before, behind = body.split("pdl_wait()")
    for word in ("after_wait(", ".load", "load<", "DT<", "__ldg", "atomic", "tma2_load", "offsets[e", "p.status ="):
        assert word not in before, word
    # every pointer that is read comes out of after_wait
    assert "after_wait(" in behind or "behind_wait()" in behind
    assert "__restrict__" not in body and "__ldg(" not in body


def test_arguments_of_the_combine_are_taken_behind_the_wait():
    text = source("token_sort.cuh")
    body = text[text.index("void behind_wait()"):]
    body = body[:body.index("}")]
    assert sorted(re.findall(r"(\w+) = after_wait\(\1\)", body)) == ["indices", "row_of", "rows", "weights"]


def test_waits_of_the_pairs_have_one_outcome():
    """Every wait of int8_pair_kernel is a whole warp's, and one that gave up still meets the others in the cluster's barriers."""
    body = kernel(source("int8_gemm.cuh"), "int8_pair_kernel")
    waits = re.findall(r"\b(mbar_wait\w*)\(", body)
    assert len(waits) == 5 and set(waits) == {"mbar_wait_warp"}
    # the epilogue of a shared tile meets twice, whether or not its wait ended well, and so do the other warps
    shared = body[body.index("if (splits > 1) {"):body.index("break;", body.index("cluster_sync_all();", body.index("if (splits > 1) {")))]
    assert shared.count("cluster_sync_all();") == 2
    for sync in re.finditer(r"cluster_sync_all\(\);", shared):
        head = shared[:sync.start()]
        assert head.count("{") - head.count("}") == 1        # not inside a condition of its own
    others = body[body.index("if (splits > 1 && (warp < 2"):]
    assert others[:others.index("}")].count("cluster_sync_all();") == 2
    # commits are awaited before a CTA ends
    assert len(re.findall(r"mbar_wait_warp\(smem_u32\(&bar_empty\[", body)) == 2


def numbers(text, name):
    return int(re.search(r"constexpr int %s = (\d+);" % name, text).group(1))


def test_the_ring_fits_beside_the_tables():
    """Groups of k-blocks by width, and shared memory with 1024 experts: 227 KB less the static arrays."""
    def block(width):
        return 128 * 128 + (width + 63) // 64 * 4096
    ring = 10 * block(64)
    for width in range(32, 257, 32):
        groups = ring // (2 * block(width))
        assert 3 <= groups <= 5 and 2 * groups * block(width) <= ring
        half = width // 2                       # rows of tokens that a CTA copies: boxes of 32, or one of 128
        boxes = 4 if half > 96 else -(-half // 32)
        assert half <= 32 * boxes and 128 * 128 + boxes * 4096 <= block(width)
        for splits in (2, 3, 4):                # sums that meet in the ring's place
            slots = {(c // splits * splits + part) for c in range(width // 32) for part in range(splits)}
            assert (max(slots) + 1) * 128 * 32 * 4 <= ring
    text = source("int8_gemm.cuh")
    assert "return 128 * 128 + (width + 63) / 64 * 4096;" in text and "kInt8Ring = 10 * int8_block_bytes(64)" in text
    assert ring + 1024 + 8 * 32 * 64 + 2 * 1025 * 4 + 512 <= 227 * 1024


@pytest.mark.parametrize("width", [32, 64, 128, 256])
def test_tiles_cover_all_rows(width):
    """The rows of an expert are cut into tiles of one height, a multiple of 32; none is left without rows."""
    for rows in list(range(1, 1100)) + [4095, 4096, 4097, 16383, 100003]:
        tiles = -(-rows // width)
        step = (-(-rows // tiles) + 31) & ~31
        assert step <= width and (tiles - 1) * step < rows <= tiles * step


def test_rows_of_a_column_kernel_cover_all():
    """Parts of a strip are multiples of 16 rows; none is left without rows."""
    for M in list(range(1, 3000)) + [4097, 65537]:
        parts = min(4, -(-M // 256))
        rows = (-(-M // parts) + 15) & ~15
        assert (parts - 1) * rows < M <= parts * rows
