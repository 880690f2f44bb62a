"""The Zig shim's kv_cache_of refuses what KvCache refuses in Python; there is no Zig compiler here, so its source is read."""
import re

from test_zig_shim import SHIM


def test_keys_and_values_of_other_shapes_are_refused():
    """Equal numbers of codes are not enough: [pages, heads, page, dim] and [pages, heads, dim, page] would be read as one another."""
    body = re.search(r"^pub fn kv_cache_of\(.*?^\}", open(SHIM).read(), re.M | re.S).group(0)
    assert re.search(r"for \(k\.shape, v\.shape\) \|a, b\| if \(a != b\) return TensorMathError\.InputTensorsWrongShape;", body)
    assert body.index("InvalidRank") < body.index("for (k.shape") < body.index("return KvCacheData")
