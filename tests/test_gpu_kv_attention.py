"""kv_cache_attention against 64 bits, with bounds that follow from what is rounded where (decode_ops_reference.attention)."""
import numpy as np
import pytest

import decode_ops_reference as ref
from test_gpu_kv_cache import as_kind, ints, on_gpu, tables

pytestmark = pytest.mark.gpu


def within(got, want, off, what=""):
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]} +- {off[bad][0]}; worst ratio {np.nanmax(np.abs(got - want) / off)}"


def run(ctx, zb, torch, cache, q, table, lengths, offsets, kind, lse=True, odd=False, **kw):
    rows, heads, dim = q[0].shape
    got = on_gpu(torch, zb, cache)
    dt, dl, do = ints(torch, table, lengths, offsets)
    pad = 5 if odd else 0
    t = torch.zeros(rows, heads * dim + pad, dtype=q[1].dtype, device="cuda")[:, pad:]
    t.copy_(q[1].view(rows, heads * dim))
    out = torch.full((rows, heads * dim + pad), 7.0, dtype=q[1].dtype, device="cuda")[:, :heads * dim]
    ls = torch.full((rows, heads), 7.0, device="cuda") if lse else None
    ctx.kv_cache_attention(got, t, dt, dl, offsets=do, out=out, lse=ls, **kw)
    ctx.synchronize()
    return out.double().cpu().numpy().reshape(rows, heads, dim), None if ls is None else ls.double().cpu().numpy()


def check(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind, window=0, sinks=0, scale=None, spare=0, odd=False, seed=0, uniform=False, change=None, q_size=1.5):
    import torch
    rng = np.random.default_rng(seed + sum(lengths) + dim)
    pages = max(1, sum(-(-max(n, 0) // page) for n in lengths)) + 2
    cache = ref.Cache(pages, kv_heads, page, dim, rng)
    table = tables(rng, pages, page, [max(n, 0) for n in lengths], 1)
    offsets = None if uniform else np.concatenate([[0], np.cumsum(new)])
    q = as_kind(torch, rng.standard_normal((sum(new) + spare, heads, dim)) * q_size, kind)
    if change:
        change(cache, table, q)
        q = q[0], torch.from_numpy(q[0]).to(q[1].dtype).cuda()
    want, off, lse, lse_off, there = ref.attention(cache, q[0], table, lengths, offsets, kind, scale, window, sinks)
    assert there[:sum(new)].all() and not there[sum(new):].any()
    got, got_lse = run(ctx, zb, torch, cache, q, table, lengths, offsets, kind, scale=scale, window=window, sinks=sinks, odd=odd)
    assert (got[~there] == 7).all() and (got_lse[~there] == 7).all()
    within(got[there], want[there], off[there], "out")
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got_lse)[there], empty[there]) and (got[there][empty[there]] == 0).all()
    within(got_lse[there & ~empty.any(1)], lse[there & ~empty.any(1)], lse_off[there & ~empty.any(1)], "lse")


DECODE = [  # new tokens, lengths, heads, kv heads, dim, page
    ([1], [1], 1, 1, 16, 16), ([1], [2], 4, 2, 64, 16), ([1], [31], 8, 1, 128, 32), ([1], [32], 8, 8, 128, 16), ([1], [33], 5, 1, 80, 32),
    ([1, 1, 1], [15, 16, 17], 6, 2, 96, 16), ([1], [700], 40, 8, 128, 32), ([1, 1], [1000, 3], 16, 2, 256, 64), ([1], [777], 7, 1, 144, 128),
    ([1, 2, 3, 0, 5], [100, 2, 300, 50, 5], 12, 4, 64, 16), ([4], [513], 16, 2, 128, 256), ([2, 7], [260, 129], 24, 2, 112, 64),
    ([1], [4111], 2, 1, 128, 64), ([3, 1], [2500, 40], 10, 1, 256, 16), ([1] * 40, list(range(1, 400, 10)), 4, 1, 64, 32)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,dim,page", DECODE)
def test_few_tokens(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind):
    check(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind, spare=len(new) % 3)


PROMPTS = [
    ([40], [40], 4, 4, 64, 16), ([130], [130], 4, 2, 128, 64), ([100, 1, 0, 29], [400, 1, 10, 30], 6, 2, 96, 32), ([257], [300], 5, 1, 128, 128),
    ([33], [200], 2, 1, 256, 16), ([129, 128, 127], [129, 500, 127], 3, 1, 80, 256), ([1, 300], [600, 300], 8, 2, 128, 64), ([150], [151], 16, 2, 48, 16),
    ([200, 7], [200, 900], 7, 1, 128, 32), ([64, 64, 64], [64, 128, 1000], 12, 12, 96, 64),
    ([150, 1], [900, 200], 4, 2, 256, 32), ([130], [130], 3, 1, 144, 16), ([70, 100, 1], [70, 300, 5], 4, 4, 208, 128), ([257], [1000], 2, 2, 256, 256)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,dim,page", PROMPTS)
def test_prompts(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind):
    check(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind, spare=2)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (5, 0), (32, 4), (33, 1), (64, 64), (100, 40), (130, 200), (10 ** 6, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,dim,page", [([1, 1], [500, 90], 8, 2, 128, 16), ([3, 2, 1], [300, 100, 33], 6, 1, 64, 32), ([150, 20], [400, 20], 4, 2, 96, 64), ([300], [300], 5, 1, 128, 32), ([140], [500], 2, 1, 256, 16)])
def test_windows_and_sinks(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind, window, sinks):
    check(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind, window=window, sinks=sinks)


@pytest.mark.parametrize("seqs,kv_heads,new", [(100, 5, 1), (128, 8, 1), (129, 4, 1), (70, 8, 3), (60, 4, 12)])
def test_more_sequences_than_there_is_room_for(ctx, zb, seqs, kv_heads, new):
    """The longest go first; equal lengths, lengths of zero."""
    rng = np.random.default_rng(seqs)
    lengths = rng.integers(0, 200, seqs)
    lengths[::7] = 64
    lengths[5:9] = 0
    check(ctx, zb, [new] * seqs, list(lengths), kv_heads * 2, kv_heads, 64, 16, "bf16", uniform=True)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [2, 90])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 1e-20])
def test_scales(ctx, zb, new, scale, kind):
    check(ctx, zb, [new, new], [new, 300], 4, 2, 64, 16, kind, scale=scale, q_size=0.3)


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32 + 5, 2 ** 40])
def test_windows_beyond_int32_are_none(ctx, zb, window):
    check(ctx, zb, [2], [300], 2, 1, 64, 16, "bf16", window=window, sinks=window)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_decoding_and_prompts_in_one_call(ctx, zb, kind):
    """Both kernels run, each takes its sequences; rows of none are left as they were."""
    check(ctx, zb, [1, 300, 0, 2, 5, 130, 1, 40], [700, 300, 50, 90, 2000, 131, 1, 41], 10, 2, 128, 32, kind, spare=3)
    check(ctx, zb, [1] * 30 + [400], [100 + 7 * i for i in range(30)] + [400], 8, 4, 64, 16, kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_equal_shares_without_offsets(ctx, zb, new, kind):
    check(ctx, zb, [new] * 4, [new, 100, 2 * new, 1000], 8, 2, 128, 32, kind, uniform=True)


@pytest.mark.parametrize("new", [2, 60])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rows_at_any_address(ctx, zb, new, kind):
    check(ctx, zb, [new, 1], [90, 200], 6, 2, 80, 16, kind, odd=True, spare=1)


@pytest.mark.parametrize("new", [2, 60])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_pages_that_are_not_there(ctx, zb, new, kind):
    """Pages outside the cache are seen by no query; where all are, the result is 0."""
    def change(cache, table, q):
        table[0, 1], table[0, 3], table[1, :] = -1, cache.pages, 2 ** 31 - 1
    check(ctx, zb, [new, new, new], [200, 100, 64], 4, 2, 64, 16, kind, change=change)


@pytest.mark.parametrize("new", [5, 90])
def test_more_new_tokens_than_the_length_says(ctx, zb, new):
    """Queries at positions below zero see nothing, the others what there is."""
    check(ctx, zb, [new, new, new], [new - 3, 0, -7], 4, 2, 64, 16, "bf16")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("what", ["loud", "quiet", "steep", "flat values", "one loud page", "zero values", "zero keys"])
def test_distributions(ctx, zb, new, what, kind):
    def change(cache, table, q):
        if what == "loud":
            cache.scales[1][:] *= 1e3
            q[0][:] *= 2.0 ** 10
            cache.scales[0][:] *= 2.0 ** -10
        if what == "quiet":
            cache.scales[1][:] *= 1e-3
            q[0][:] *= 2.0 ** -12
            cache.scales[0][:] *= 2.0 ** 12
        if what == "flat values":
            cache.codes[1][:] = 100
        if what == "one loud page":
            cache.scales[1][table[0, 1]] *= 300
        if what == "zero values":
            cache.codes[1][:] = 0
            cache.scales[1][::2] = 0
        if what == "zero keys":
            cache.scales[0][:] = 0
    check(ctx, zb, [new], [new + 333], 4, 1, 128, 32, kind, change=change, q_size=12.0 if what == "steep" else 1.0)


@pytest.mark.parametrize("pages", [30, 40])      # with 30 some places of the table have no page
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_nan_stays_where_it_belongs(ctx, zb, new, kind, pages):
    """A page with a scale of NaN spoils the queries that see it, a query with a NaN or an infinity itself; masked places spoil nothing."""
    import torch
    rng = np.random.default_rng(2)
    cache = ref.Cache(pages, 2, 16, 64, rng)
    lengths = [200, 200, 150]
    table = tables(rng, 40, 16, lengths)
    table[table >= pages] = -1
    window, sinks = 40, 3
    rows = 3 * new
    first = [n - new for n in lengths]
    # out of every query's window, and behind the last token
    hidden = table[0, 4]
    cache.scales[0][hidden], cache.scales[1][hidden] = np.nan, np.nan
    q = rng.standard_normal((rows, 4, 64))
    q[new, 1, 5], q[new, 2, 7] = np.nan, np.inf                 # sequence 1, first row, heads 1 and 2
    last = table[2, 149 // 16]
    cache.scales[1][last, 0] = np.nan                          # sequence 2's last page, values of head 0
    q = as_kind(torch, q, kind)
    clean = cache.copy()
    for s in clean.scales:
        s[np.isnan(s)] = 0.01
    want, off, _, _, _ = ref.attention(clean, np.where(np.isfinite(q[0]), q[0], 0), table, lengths, None, kind, None, window, sinks)
    got, lse = run(ctx, zb, torch, cache, q, table, lengths, None, kind, window=window, sinks=sinks)
    nan = np.zeros(got.shape[:2], bool)
    nan[new, 1:3] = True
    for s, i, h in np.ndindex(3, new, 2):
        at = first[s] + i
        seen = {ref.page_of(cache, table, s, j) for j in range(at + 1) if j > at - window or j < sinks} - {-1}
        if any(np.isnan(cache.scales[kv][p, h]) for kv in range(2) for p in seen):
            nan[s * new + i, 2 * h:2 * h + 2] = True
    assert pages == 30 or nan[2 * new:].any()
    assert np.array_equal(np.isnan(got).all(2), nan) and np.array_equal(np.isnan(got).any(2), nan)
    within(got[~nan], want[~nan], off[~nan])


def test_a_cache_beyond_32_bits(ctx, zb):
    """Pages at the end of a cache of more than 2^32 bytes of codes."""
    import torch
    rng = np.random.default_rng(9)
    small = ref.Cache(8, 4, 256, 256, rng)
    pages = (1 << 32) // (4 * 256 * 256) + 40
    k, v = (torch.zeros(pages, 4, 256, 256, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, 4, device="cuda") for _ in range(2))
    for big, part in ((k, small.codes[0]), (v, small.codes[1]), (ks, small.scales[0]), (vs, small.scales[1])):
        big[-8:] = torch.from_numpy(part).cuda()
    table = rng.permutation(8).reshape(2, 4).astype(np.int32)
    far = table + pages - 8
    for new, heads in ((2, 8), (70, 4)):
        q = as_kind(torch, rng.standard_normal((2 * new, heads, 256)), "bf16")
        want, off, _, _, _ = ref.attention(small, q[0], table, [1000, 300], None, "bf16")
        out = torch.empty(2 * new, heads, 256, dtype=torch.bfloat16, device="cuda")
        dt, dl = ints(torch, far, [1000, 300])
        cache = zb.KvCache(k, ks, v, vs)
        ctx.kv_cache_attention(cache, q[1], dt, dl, out=out)
        ctx.synchronize()
        within(out.double().cpu().numpy(), want, off)
    x = torch.randn(2, 4 * 256, device="cuda")
    ctx.kv_cache_write(cache, x, x, dt, dl)
    back = tuple(torch.empty(2, 4 * 256, device="cuda") for _ in range(2))
    ctx.kv_cache_read(cache, dt, dl, out=back)
    ctx.synchronize()
    page = k[int(far[0, 3]), 0, 999 % 256].float() * ks[int(far[0, 3]), 0]
    assert torch.equal(back[0][0, :256], page) and torch.equal(back[1], back[1])


def test_results_do_not_change_from_call_to_call(ctx, zb):
    import torch
    rng = np.random.default_rng(4)
    cache = ref.Cache(300, 2, 32, 128, rng)
    table = tables(rng, 300, 32, [4000, 3000, 1])
    q = as_kind(torch, rng.standard_normal((3 * 2, 8, 128)), "bf16")
    first = run(ctx, zb, torch, cache, q, table, [4000, 3000, 2], None, "bf16")
    for _ in range(3):
        again = run(ctx, zb, torch, cache, q, table, [4000, 3000, 2], None, "bf16")
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


def test_host_arrays(ctx, zb):
    rng = np.random.default_rng(6)
    cache = ref.Cache(10, 2, 16, 32, rng)
    table = tables(rng, 10, 16, [70, 40])
    q = rng.standard_normal((5, 4 * 32)).astype(np.float32)
    want, off, lse, lse_off, _ = ref.attention(cache, q.astype(np.float64).reshape(5, 4, 32), table, [70, 40], [0, 4, 5], "f32")
    held = zb.KvCache(*[x.copy() for x in (cache.codes[0], cache.scales[0], cache.codes[1], cache.scales[1])])
    ls = np.zeros((5, 4), np.float32)
    got = ctx.kv_cache_attention(held, q, table, [70, 40], offsets=[0, 4, 5], lse=ls)
    within(got.reshape(5, 4, 32).astype(np.float64), want, off)
    within(ls.astype(np.float64), lse, lse_off)


@pytest.mark.parametrize("new,length,dim", [(300, 600, 128), (2, 600, 128), (1, 20000, 128), (200, 300, 256)])
@pytest.mark.parametrize("cta", [0, 3, 10007])
def test_a_cta_gives_up(ctx, zb, new, length, dim, cta):
    """A CTA whose first wait runs out: every warp of it comes to the kernel's end (and its cluster), the call reports the time-out, and the calls behind it are right."""
    import torch
    rng = np.random.default_rng(8)
    cache = ref.Cache(2 * (length // 64 + 1), 2, 64, dim, rng)
    table = tables(rng, cache.pages, 64, [length, length // 2])
    q = as_kind(torch, rng.standard_normal((2 * new, 4, dim)), "bf16")
    args = (ctx, zb, torch, cache, q, table, [length, length // 2], None, "bf16")
    want = run(*args)
    ctx.selftest_give_up(cta)
    with pytest.raises(zb.ZantError) as e:
        run(*args)
    assert e.value.name == "DeviceTimeout"
    for _ in range(2):
        got = run(*args)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


LONG = [([1], [20000], 8, 2, 64, 16, "bf16"), ([1], [33000], 4, 1, 128, 32, "f16"), ([3], [17001], 16, 1, 128, 64, "bf16"), ([1], [16400], 3, 1, 80, 128, "f32"), ([1, 2], [40000, 100], 5, 1, 96, 256, "bf16"),
        ([1], [18000], 2, 1, 256, 32, "f16"), ([2], [25000], 8, 1, 112, 16, "f32")]


@pytest.mark.parametrize("new,lengths,heads,kv_heads,dim,page,kind", LONG)
def test_long_contexts_with_and_without_a_workspace(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind):
    """Few tiles of long contexts go through the arena; a context whose arena must not grow has its clusters."""
    check(ctx, zb, new, lengths, heads, kv_heads, dim, page, kind)
    assert ctx.last_kernel() == "kv_attention_join_kernel"
    tight = zb.Context(0, arena_bytes=4096)
    try:
        tight.set_arena_limit(4096)
        check(tight, zb, new, lengths, heads, kv_heads, dim, page, kind)
        assert tight.last_kernel() == "kv_attention_kernel"
    finally:
        tight.close()
