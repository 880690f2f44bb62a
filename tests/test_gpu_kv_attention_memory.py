"""kv_cache_attention over long contexts where the device has no memory for its workspace, and where a limit has: the call runs, on clusters or with a workspace."""
import pytest

from test_gpu_kv_attention import check

pytestmark = pytest.mark.gpu
CASE = ([2], [20000], 4, 1, 64, 32, "bf16")


def test_no_memory_for_the_workspace(zb):
    c = zb.Context(0, arena_bytes=4096)
    try:
        check(c, zb, *CASE)
        assert c.last_kernel() == "kv_attention_join_kernel"
    finally:
        c.close()
    c = zb.Context(0, arena_bytes=4096)
    try:
        zb.debug_fail_alloc(1)
        check(c, zb, *CASE)
        assert c.last_kernel() == "kv_attention_kernel"
        check(c, zb, *CASE)                           # there is memory again
        assert c.last_kernel() == "kv_attention_join_kernel"
    finally:
        zb.debug_fail_alloc(0)
        c.close()


@pytest.mark.parametrize("limit,kernel", [(1 << 20, "kv_attention_kernel"), (64 << 20, "kv_attention_join_kernel")])
def test_a_limit_that_the_arena_has_not_reached(zb, limit, kernel):
    c = zb.Context(0, arena_bytes=4096)
    try:
        c.set_arena_limit(limit)
        check(c, zb, *CASE)
        assert c.last_kernel() == kernel
    finally:
        c.close()
