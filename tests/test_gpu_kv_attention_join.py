"""Few tiles over long contexts, whose CTAs leave their sums in the workspace for a second kernel to join: every row of a tile is joined, and no row of a sequence that the prompts' kernel has taken."""
import numpy as np
import pytest

from test_gpu_kv_attention import check

pytestmark = pytest.mark.gpu


def fill_arena(ctx):
    """16 MB of NaN in the arena, where the next call's workspace lies."""
    import torch
    torch.cuda.synchronize()
    ctx.quantize_rows(np.full((1024, 4096), np.nan, np.float32))


ROWS = [  # 17 to 24 rows of a key head: tiles of 24
    ([17], [16500], 1, 1, 16, 64, True), ([4], [20000], 5, 1, 64, 16, True), ([3], [17000], 8, 1, 48, 32, False), ([4], [20000], 40, 8, 64, 16, False), ([23], [16385], 2, 2, 64, 128, True),
    ([3, 3], [20000, 700], 8, 1, 64, 16, True), ([5, 2, 5], [17000, 20000, 40], 5, 1, 32, 256, False), ([4], [18000], 12, 2, 128, 64, True), ([6], [17000], 3, 1, 96, 16, False)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,dim,page,uniform", ROWS)
def test_every_row_of_a_tile(ctx, zb, new, lengths, heads, kv_heads, dim, page, uniform, kind):
    fill_arena(ctx)
    check(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind, uniform=uniform)
    assert ctx.last_kernel() == "kv_attention_join_kernel"


MIXED = [  # a short prompt beside sequences with few new tokens
    ([25, 1], [300, 20000], 8, 1, 128, 32), ([1, 30, 1], [17000, 30, 200], 8, 1, 128, 64), ([10, 28], [17000, 500], 8, 1, 128, 16), ([38, 2], [40, 33000], 8, 1, 64, 128),
    ([60, 1], [100, 20000], 4, 1, 64, 16), ([1, 15], [20000, 15], 16, 1, 96, 32), ([200, 10], [200, 18000], 1, 1, 80, 256)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,dim,page", MIXED)
def test_prompts_beside_long_contexts(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind):
    fill_arena(ctx)
    check(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind, spare=2)
    assert ctx.last_kernel() == "kv_attention_join_kernel"
