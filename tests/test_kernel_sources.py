"""Rules on the kernels' sources that no run can show to be broken: what the compiler happens to place well works anyway."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "h3metal_b200", "csrc")


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def functions(text):
    """{name: body} of the device functions of ptx.cuh."""
    found = {}
    for m in re.finditer(r"__device__ __forceinline__ [\w ]+?(\w+)\(([^)]*)\) \{", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        found[m.group(1)] = text[m.end():i - 1]
    return found


def test_aligned_instructions_bring_their_warp_together_first():
    """An instruction marked .aligned is undefined for a warp whose threads are apart, as they may be behind a loop that one
    lane ran alone: its wrapper starts with __syncwarp(). The reads of tensor memory are left to their callers."""
    aligned = {n: b for n, b in functions(source("ptx.cuh")).items() if ".aligned" in b and not n.startswith("tmem_ld")}
    assert {"tmem_alloc", "tmem_dealloc", "tmem_alloc_pair", "tmem_dealloc_pair", "cluster_sync_all"} <= set(aligned)
    for name, body in aligned.items():
        assert body.strip().startswith("__syncwarp();"), name


@pytest.mark.parametrize("name", ["gemm_f8_small.cu", "gemm_f8_pair.cu"])
def test_epilogue_warps_read_tensor_memory_together(name):
    text = source(name)
    waits = [m.end() for m in re.finditer(r"ok = mbar_wait\(done_bar\(pos\.s\), pos\.ph, cta_abort", text)]
    assert waits
    for at in waits:
        assert "__all_sync(0xFFFFFFFFu, ok)" in text[at:text.index("tmem_ld_32x32b", at)]


def test_the_few_row_kernel_meets_its_barriers_with_whole_warps():
    text = source("gemm_f8_small.cu")
    for m in re.finditer(r"__syncthreads\(\);", text):
        assert text[:m.start()].rstrip().endswith("__syncwarp();")


@pytest.mark.parametrize("name", ["gemm_f8_small.cu", "gemm_f8_pair.cu"])
def test_scales_are_read_by_ordinary_loads(name):
    """The product may start while the kernel that writes its activations' scales still runs: the read-only path is not defined
    for such memory. ptx.cuh's ld_f32 is a volatile statement: it stays behind grid_dep_wait()."""
    text = source(name)
    assert "__ldg" not in text and "ld.global.nc" not in text and text.count("ld_f32(") >= 3
    body = functions(source("ptx.cuh"))["ld_f32"]
    assert "asm volatile" in body and "ld.global.f32" in body


@pytest.mark.parametrize("name", ["gemm_f8_small.cu", "gemm_f8_pair.cu"])
def test_the_issuer_waits_for_its_instructions_when_a_wait_ran_out(name):
    """Between the issuing loop and the end of the issuer's branch: a bounded wait on the stage that was committed last."""
    text = source(name)
    tail = text[text.index("umma_commit"):]
    tail = tail[:tail.index("tmem_dealloc")]
    assert re.search(r"if \(\*cta_abort && issued\) \{\s*pos\.retreat\(stages\);\s*int dummy_abort = 0;\s*"
                     r"mbar_wait\(done_bar\(pos\.s\), pos\.ph, &dummy_abort", tail)


@pytest.mark.parametrize("name", ["gemm_w8a8.cu", "gemm_w8a8_pair.cu"])
def test_the_int8_product_reads_its_activations_scales_the_same_way(name):
    text = source(name)
    assert "ld_f32(g.sa" in text and not re.search(r"__ldg\(g\.sa\b", text)
