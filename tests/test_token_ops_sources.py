"""Rules of the language-model kernels whose breach shows in no result for certain: read from their sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "z-ant_b200", "csrc")


def source(name):
    """The file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_barriers_that_other_ctas_arrive_on_are_waited_for_at_cluster_scope():
    text = source("scaled_gemm_q8.cuh")
    pair = text[text.index("scaled_pair_kernel(const __grid_constant__"):text.index("struct ScaledFew")]
    remote = set(re.findall(r"mbar_arrive_cluster\(ptx::cluster_addr\(bar\.(\w+)\(", text))
    assert remote == {"tempty"}
    for name in remote:
        waits = re.findall(r"(\w+(?:<\w+>)?)\((?:a, )?bar\.%s\([^;]*abort_flag" % name, pair)
        assert waits and all(w.endswith("<true>") for w in waits), waits
    ptx = source("ptx_sm100.cuh")
    assert "mbarrier.try_wait.parity.acquire.cluster" in ptx and "mbarrier.arrive.release.cluster" in ptx


def test_what_the_kernel_before_may_write_is_read_by_coherent_loads():
    """These kernels start beside the one that writes their operands: no load among them is a non-coherent one."""
    for name in ("quantize_rows.cuh", "scaled_gemm_q8.cuh", "token_logprobs.cuh"):
        text = source(name)
        assert "grid_start()" in text or "grid_wait()" in text
        assert not re.findall(r"__ldg\(|ld_global_nc|\.nc\.", text), name
    once = source("ptx_sm100.cuh")
    once = once[once.index("uint4 ld_global_once("):]
    assert "asm volatile" in once[:once.index("}")] and ".nc" not in once[:once.index("}")]


def test_lanes_come_together_in_front_of_instructions_of_the_whole_warp():
    """tcgen05.ld, mma.sync and barrier.cluster are executed by all lanes of a warp at once: behind stores, loads or branches of single lanes stands a warp barrier."""
    gemm, logp = source("scaled_gemm_q8.cuh"), source("token_logprobs.cuh")
    epilogue = gemm[gemm.index("tmem_ld32("):gemm.index("tc_fence_before", gemm.index("tmem_ld32("))]
    assert re.search(r"store_columns_any\([^;]*;\s*if \(!all_live\) __syncwarp\(\);\s*\}", epilogue)
    step = gemm[gemm.index("auto step = [&](int c, bool all)"):gemm.index("mma_m16n8k32_s8(")]
    assert re.search(r"if \(ANY \|\| !all\) __syncwarp\(\);", step)
    for m in re.finditer(r"cluster_arrive\(\)", logp):
        assert re.search(r"__syncwarp\(\);\s*(if \(P > 1\) )?ptx::$", logp[:m.start()])
