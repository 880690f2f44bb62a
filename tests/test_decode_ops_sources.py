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
