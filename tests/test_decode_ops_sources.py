"""Rules of the kernels on a decoder's int8 cache whose breach shows in no result for certain: read from their sources."""
import re

from test_token_ops_sources import source


def test_the_ring_of_copies_is_written_by_copies_alone():
    """Until the last copy has landed (the sums come then), the shared memory that TMA fills is only read: a plain store in front of a copy would need a fence of proxies."""
    text = source("kv_attention.cuh")
    kernel = text[text.index("kv_attention_kernel(const __grid_constant__"):]
    kernel = kernel[:kernel.index("float* sums = reinterpret_cast<float*>(smem)")]
    assert set(re.findall(r"(\w+)\*\s+\w+\s*=\s*(?:reinterpret_cast<[^>]*>\()?smem\b(?!\s*\+\s*F::big)", kernel)) == {"uint8_t"}      # (one pointer: the ring, of const bytes)
    assert re.search(r"const uint8_t\* ring = smem \+", kernel)
    assert len(re.findall(r"\bsmem\b", kernel)) == len(re.findall(r"\bsmem \+ F::big\(W\)", kernel)) + 2       # its declaration, the ring


def test_lanes_come_together_in_front_of_instructions_of_the_whole_warp():
    """tcgen05.ld and bar.sync are executed by all lanes of a warp at once: behind stores of single lanes stands a warp barrier."""
    text = source("kv_prompt.cuh")
    rows = text[text.index("void kv_prompt_rows("):text.index("kv_prompt_kernel(const __grid_constant__")]
    end = rows[rows.index("float out_scale"):]
    assert re.search(r"uint32_t v\[16\];\s*__syncwarp\(\);\s*if \(count > 0\) \{\s*ptx::tmem_ld16\(", end) and end.count("tmem_ld16(") == 1
    for m in re.finditer(r"named_barrier_sync\(", text):
        assert re.search(r"__syncwarp\(\);\s*ptx::$", text[:m.start()])
