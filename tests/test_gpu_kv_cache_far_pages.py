"""kv_cache_write and kv_cache_read on pages at the end of a cache of more than 2^32 bytes of codes: scales, codes and rows to the bit, and nothing elsewhere is touched."""
import numpy as np
import pytest

import decode_ops_reference as ref
from test_gpu_kv_cache import as_kind, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,new", [("f32", 2), ("bf16", 1), ("bf16", 300), ("f32", 256)])
def test_write_and_read(ctx, zb, kind, new):
    import torch
    rng = np.random.default_rng(new)
    heads, page, dim = 4, 256, 256
    small = ref.Cache(8, heads, page, dim, rng)
    pages = (1 << 32) // (heads * page * dim) + 40
    big = [torch.zeros(pages, heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)], [torch.zeros(pages, heads, device="cuda") for _ in range(2)]
    for kv in range(2):
        big[0][kv][-8:], big[1][kv][-8:] = torch.from_numpy(small.codes[kv]).cuda(), torch.from_numpy(small.scales[kv]).cuda()
    table = rng.permutation(8).reshape(2, 4).astype(np.int32)
    lengths = [1000, 301]
    x = [as_kind(torch, rng.standard_normal((2 * new, heads * dim)) * 3, kind) for _ in range(2)]
    dt, dl = ints(torch, table + (pages - 8), lengths)
    cache = zb.KvCache(big[0][0], big[1][0], big[0][1], big[1][1])
    ctx.kv_cache_write(cache, x[0][1], x[1][1], dt, dl)
    out = tuple(torch.full((2 * new, heads * dim), 5.0, dtype=x[0][1].dtype, device="cuda") for _ in range(2))
    ctx.kv_cache_read(cache, dt, dl, out=out)
    ctx.synchronize()
    ref.write(small, [a.reshape(-1, heads, dim) for a, _ in x], table, lengths, None)
    for kv in range(2):
        assert not big[0][kv][:-8].any() and not big[1][kv][:-8].any()
        assert np.array_equal(big[0][kv][-8:].cpu().numpy(), small.codes[kv]) and np.array_equal(big[1][kv][-8:].cpu().numpy(), small.scales[kv])
        want, there = ref.read(small, kv, 2 * new, table, lengths, None)
        assert there.all()
        # code * scale is rounded to fp32 and from there to the type
        want = torch.from_numpy(want.astype(np.float32)).to(out[kv].dtype).view(2 * new, heads * dim)
        assert torch.equal(out[kv].cpu(), want)
