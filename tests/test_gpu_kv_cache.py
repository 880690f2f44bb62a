"""kv_cache_write and kv_cache_read against their plain forms: codes, scales and what comes back, to the bit."""
import numpy as np
import pytest

import decode_ops_reference as ref

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "bf16"]


def as_kind(torch, x, kind):
    """float64 -> (values as the type has them, torch tensor on the GPU)."""
    t = torch.from_numpy(x).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind])
    return t.double().numpy(), t.cuda()


def on_gpu(torch, zb, cache):
    """The package's form of a reference cache: arrays on the GPU."""
    t = [torch.from_numpy(x.copy()).cuda() for x in (cache.codes[0], cache.scales[0], cache.codes[1], cache.scales[1])]
    return zb.KvCache(*t)


def same(cache, got):
    for kv, (codes, scales) in enumerate(((got.k, got.k_scale), (got.v, got.v_scale))):
        codes, scales = (a if isinstance(a, np.ndarray) else a.cpu().numpy() for a in (codes, scales))
        assert np.array_equal(scales, cache.scales[kv], equal_nan=True), kv
        assert np.array_equal(codes, cache.codes[kv]), kv


def tables(rng, pages, page, lengths, extra=0):
    """Distinct pages for every sequence, -1 behind the last."""
    wide = [-(-n // page) for n in lengths]
    width = max(wide + [1]) + extra
    order = rng.permutation(pages)
    table, at = np.full((len(lengths), width), -1, np.int32), 0
    for s, w in enumerate(wide):
        table[s, :w] = order[at:at + w]
        at += w
    assert at <= pages
    return table


def ints(torch, *arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda() for a in arrays]


CASES = [  # new tokens, lengths, heads, page, dim
    ([1], [1], 1, 16, 16), ([1], [16], 2, 16, 64), ([1], [17], 3, 16, 48), ([5], [33], 2, 32, 80), ([1, 1, 1], [31, 32, 33], 2, 32, 128),
    ([64], [64], 2, 64, 128), ([300], [300], 1, 64, 96), ([70, 1, 0, 130], [70, 255, 40, 400], 2, 64, 256), ([257], [1000], 1, 256, 32), ([3, 40], [200, 41], 5, 128, 112)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,lengths,heads,page,dim", CASES)
@pytest.mark.parametrize("odd", [False, True])
def test_write_and_read(ctx, zb, new, lengths, heads, page, dim, kind, odd):
    import torch
    rng = np.random.default_rng(sum(lengths) + dim)
    pages = sum(-(-n // page) for n in lengths) + 3
    cache = ref.Cache(pages, heads, page, dim, rng)
    table = tables(rng, pages, page, lengths, 2)
    offsets = np.concatenate([[0], np.cumsum(new)])
    rows, spare = sum(new), 3
    x = [as_kind(torch, rng.standard_normal((rows + spare, heads * dim)) * np.exp(rng.standard_normal((rows + spare, 1))), kind) for _ in range(2)]
    got = on_gpu(torch, zb, cache)
    dt, dl, do = ints(torch, table, lengths, offsets)
    if odd:                                         # rows at any address, further apart than they are long
        room = [torch.zeros(rows + spare, heads * dim + 7, dtype=x[0][1].dtype, device="cuda") for _ in range(2)]
        k, v = (r[:, 1:1 + heads * dim] for r in room)
        k.copy_(x[0][1]); v.copy_(x[1][1])
    else:
        k, v = x[0][1], x[1][1].view(rows + spare, heads, dim)
    ctx.kv_cache_write(got, k, v, dt, dl, offsets=do)
    ctx.synchronize()
    ref.write(cache, [a.reshape(-1, heads, dim) for a, _ in x], table, lengths, offsets)
    same(cache, got)
    # all of each sequence back, and rows that belong to none
    total = sum(lengths)
    oo = np.concatenate([[0], np.cumsum(lengths)])
    out = [torch.full((total + spare, heads * dim + (7 if odd else 0)), 5.0, dtype=x[0][1].dtype, device="cuda")[:, (1 if odd else 0):][:, :heads * dim] for _ in range(2)]
    ctx.kv_cache_read(got, dt, dl, offsets=ints(torch, oo)[0], out=tuple(out))
    ctx.synchronize()
    for kv in range(2):
        want, there = ref.read(cache, kv, total + spare, table, lengths, oo)
        assert there[:total].all() and not there[total:].any()
        # code * scale is rounded to fp32 and from there to the type
        want = torch.from_numpy(want.astype(np.float32)).to(x[0][1].dtype).float().numpy().reshape(total + spare, -1)
        want[total:] = 5.0
        assert np.array_equal(out[kv].float().cpu().numpy(), want)


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_one_by_one(ctx, zb, kind):
    """A sequence that grows by one token a call, louder and quieter ones: each page's scale grows and its codes follow."""
    import torch
    rng = np.random.default_rng(7)
    cache = ref.Cache(4, 2, 16, 32, rng)
    got = on_gpu(torch, zb, cache)
    table = np.array([[2, 0, 3]], np.int32)
    dt, = ints(torch, table)
    for n in range(1, 40):
        x = [as_kind(torch, rng.standard_normal((1, 64)) * np.exp(2 * rng.standard_normal()) * (0.0 if n % 13 == 5 else 1.0), kind) for _ in range(2)]
        ctx.kv_cache_write(got, x[0][1], x[1][1], dt, ints(torch, [n])[0])
        ctx.synchronize()
        ref.write(cache, [a.reshape(1, 2, 32) for a, _ in x], table, [n], None)
        same(cache, got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", ["tiny", "huge", "ties", "zero", "nan", "inf"])
def test_values_at_the_ends(ctx, zb, kind, size):
    import torch
    rng = np.random.default_rng(11)
    cache = ref.Cache(3, 1, 32, 64, rng)
    for s in cache.scales:
        s[:] = {"tiny": 1e-38 if kind != "f16" else 1e-7, "huge": 1.0, "zero": 0.0}.get(size, 0.01)
    table = np.array([[1, 2]], np.int32)
    x = rng.standard_normal((40, 64))
    if size == "tiny":
        x *= 3e-38 if kind != "f16" else 6e-7
    if size == "huge":
        x *= 1e37 if kind != "f16" else 15000
    if size == "ties":
        x = rng.integers(-254, 255, (40, 64)) / 2.0
        x[0, 0] = x[20, 0] = 127.0
    if size == "zero":
        x[:] = 0
    if size in ("nan", "inf"):
        x[3, 5] = float(size)
    v = as_kind(torch, x, kind)
    got = on_gpu(torch, zb, cache)
    dt, dl = ints(torch, table, [47])
    for _ in range(2):                              # begun pages, and the same again
        ctx.kv_cache_write(got, v[1], v[1], dt, dl)
        ctx.synchronize()
        ref.write(cache, [v[0].reshape(40, 1, 64)] * 2, table, [47], None)
        same(cache, got)


def test_pages_outside_and_lengths_that_do_not_fit(ctx, zb):
    """Nothing is written for pages outside the cache, positions below zero and beyond the table; reads give zeros there."""
    import torch
    rng = np.random.default_rng(5)
    cache = ref.Cache(6, 2, 16, 32, rng)
    table = np.array([[0, -1, 1], [7, 2, 2 ** 31 - 1], [3, 4, 5], [-2 ** 31, 6, -1]], np.int32)
    lengths, offsets = [40, 1000, 3, 20], [0, 30, 40, 50, 60]
    x = [as_kind(torch, rng.standard_normal((64, 64)), "f32") for _ in range(2)]
    got = on_gpu(torch, zb, cache)
    dt, dl, do = ints(torch, table, lengths, offsets)
    ctx.kv_cache_write(got, x[0][1], x[1][1], dt, dl, offsets=do)
    ctx.synchronize()
    ref.write(cache, [a.reshape(64, 2, 32) for a, _ in x], table, lengths, offsets)
    same(cache, got)
    out = tuple(torch.full((64, 64), 5.0, device="cuda") for _ in range(2))
    ctx.kv_cache_read(got, dt, dl, offsets=do, out=out)
    ctx.synchronize()
    for kv in range(2):
        want, there = ref.read(cache, kv, 64, table, lengths, offsets)
        want = np.where(there[:, None], want.astype(np.float32).reshape(64, 64), 5.0)
        assert np.array_equal(out[kv].cpu().numpy(), want)


@pytest.mark.parametrize("seqs", [33, 200, 1100])
def test_many_sequences(ctx, zb, seqs):
    """The search for a page's sequence: many of them, some with nothing new."""
    import torch
    rng = np.random.default_rng(seqs)
    new = rng.integers(0, 4, seqs) * rng.integers(0, 2, seqs) + (rng.random(seqs) < 0.01) * 40
    lengths = new + rng.integers(0, 40, seqs)
    pages = int(sum(-(-n // 16) for n in lengths))
    cache = ref.Cache(pages, 1, 16, 16, rng)
    table = tables(rng, pages, 16, list(lengths))
    offsets = np.concatenate([[0], np.cumsum(new)])
    x = [as_kind(torch, rng.standard_normal((int(new.sum()), 16)), "bf16") for _ in range(2)]
    got = on_gpu(torch, zb, cache)
    dt, dl, do = ints(torch, table, lengths, offsets)
    ctx.kv_cache_write(got, x[0][1], x[1][1], dt, dl, offsets=do)
    ctx.synchronize()
    ref.write(cache, [a.reshape(-1, 1, 16) for a, _ in x], table, lengths, offsets)
    same(cache, got)


@pytest.mark.parametrize("offsets", [[0, 9, 4, 12], [5, 2, 1, 0], [-4, 3, 30, 7], [12, 12, 0, 12], [0, 0, 0, 0]])
def test_offsets_out_of_order_stay_inside(ctx, zb, offsets):
    """Which rows a sequence has is not defined then, but nothing outside its own pages changes."""
    import torch
    rng = np.random.default_rng(3)
    cache = ref.Cache(8, 1, 16, 16, rng)
    got = on_gpu(torch, zb, cache)
    table = np.array([[0, 1], [2, 3], [4, -1]], np.int32)
    x = torch.ones(12, 16, device="cuda")
    dt, dl, do = ints(torch, table, [20, 32, 9], offsets)
    ctx.kv_cache_write(got, x, x, dt, dl, offsets=do)
    ctx.synchronize()
    for codes, scales, c, s in ((got.k, got.k_scale, cache.codes[0], cache.scales[0]), (got.v, got.v_scale, cache.codes[1], cache.scales[1])):
        assert np.array_equal(codes.cpu().numpy()[5:], c[5:]) and np.array_equal(scales.cpu().numpy()[5:], s[5:])


def test_host_arrays(ctx, zb):
    rng = np.random.default_rng(1)
    cache = ref.Cache(9, 2, 16, 48, rng)
    got = zb.KvCache(cache.codes[0].copy(), cache.scales[0].copy(), cache.codes[1].copy(), cache.scales[1].copy())
    lengths, offsets = [20, 50], [0, 20, 31]
    table = tables(rng, 9, 16, lengths)
    x = [rng.standard_normal((31, 96)).astype(np.float16) for _ in range(2)]
    ctx.kv_cache_write(got, x[0], x[1].reshape(31, 2, 48), table, lengths, offsets=offsets)
    ref.write(cache, [a.astype(np.float64).reshape(31, 2, 48) for a in x], table, lengths, offsets)
    same(cache, got)
    k, v = ctx.kv_cache_read(got, table, lengths, offsets=[0, 20, 70], rows=70)
    for kv, y in enumerate((k, v)):
        assert np.array_equal(y, ref.read(cache, kv, 70, table, lengths, [0, 20, 70])[0].reshape(70, 96).astype(np.float32))
    only = np.zeros((70, 2, 48), np.float16)
    ctx.kv_cache_read(got, table, lengths, offsets=[0, 20, 70], out=(None, only))
    assert np.array_equal(only.reshape(70, 96), v.astype(np.float16))
    ctx.kv_cache_read(got, table, lengths, offsets=[0, 20, 70], out=(only, None))
    assert np.array_equal(only.reshape(70, 96), k.astype(np.float16))
