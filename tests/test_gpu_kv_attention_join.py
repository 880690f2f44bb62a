"""Few tiles over long contexts, whose CTAs leave their sums in the workspace for a second kernel to join: every row of a tile is joined."""
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
