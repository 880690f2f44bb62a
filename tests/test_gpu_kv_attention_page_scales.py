"""kv_cache_attention where pages' scales of V lie far apart: a row's result is as exact, relative to the largest weight times scale that it sees itself, as where they are alike."""
import numpy as np
import pytest

import decode_ops_reference as ref
from test_gpu_kv_attention import run, within
from test_gpu_kv_cache import as_kind, tables

pytestmark = pytest.mark.gpu
U = ref.U


def attention(cache, q, table, length, new, kind, scale, window, sinks):
    """(out, how far off it may be, what that adds to lse's) of one sequence's last rows.

    decode_ops_reference.attention has the terms of scores, weights and sums.  Three differ here.  What f16 loses of a weight below its least numbers is half of 2^-24 where the row's largest weight times
    scale is 2^6 at least: 2^-31 of that one for each token, times a code of 127 at most.  Powers of two of exponents up to L + X in magnitude (the binary logarithms of the scales' ratios, and of the weights) come from
    fp32 numbers that are off by a few of their half steps, 16 U (L + X + 8) in all, and with them each weight, the sum of them and what the row is multiplied with at the end.  And f32's two f16 numbers of a weight lose no more than 2^-31 of that largest one
    either."""
    rows, heads, dim = q.shape
    group = heads // cache.heads
    scale = dim ** -0.5 if scale is None else scale
    out, off, more = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, heads))
    pos = np.arange(length)
    where, slot = table[0, pos // cache.page], pos % cache.page
    for h in range(cache.heads):
        vs = cache.scales[1][where, h].astype(np.float64)
        k = cache.codes[0][where, h, slot].astype(np.float64) * cache.scales[0][where, h].astype(np.float64)[:, None]
        v = cache.codes[1][where, h, slot].astype(np.float64) * vs[:, None]
        for i in range(new):
            at = length - new + i
            j = np.flatnonzero((pos <= at) & ((window == 0) | (pos > at - window) | (pos < sinks)))
            for g in range(h * group, (h + 1) * group):
                x = (k[j] @ q[i, g]) * scale
                size = (np.abs(k[j]) @ np.abs(q[i, g])) * abs(scale)
                e = np.exp(x - x.max())
                w = e / e.sum()
                out[i, g] = w @ v[j]
                dx = (2 * U * (dim + 2) * size + (2.0 ** -27 if kind == "f32" else 2.0 ** -20) * abs(scale) * np.abs(q[i, g]).max() * np.abs(k[j]).sum(1)).max()
                some = vs[j][vs[j] > 0]
                far = 0.0 if kind == "f32" or not len(some) else 16 * U * (np.log2(vs.max() / some.min()) + np.abs(x).max() * 1.45 + 8)
                dw = 2 * (dx + 8 * U + 6 * U * np.abs(x - x.max())) + far
                more[i, g] = far
                h16 = 2.0 ** -22 if kind == "f32" else 2.0 ** -11
                wide = 2 * U * (len(j) / 4 + 64)
                mean = w @ np.abs(v[j])
                o = (w * (dw + h16)) @ np.abs(v[j]) + mean * (w @ dw + 2 * wide + far) + 2.0 ** -31 * (w * vs[j]).max() * 127 * len(j)
                off[i, g] = o + ref.HALF_STEP[kind] * (np.abs(out[i, g]) + o) + ref.LEAST[kind]
    return out, off, more


def compare(ctx, zb, new, length, heads, kv_heads, dim, page, kind, change, window=0, sinks=0, scale=None):
    import torch
    rng = np.random.default_rng(length + dim + new)
    cache = ref.Cache(-(-length // page) + 1, kv_heads, page, dim, rng)
    table = tables(rng, cache.pages, page, [length])
    q = rng.standard_normal((new, heads, dim))
    change(cache, table[0], q)
    q = as_kind(torch, q, kind)
    want, off, more = attention(cache, q[0], table, length, new, kind, scale, window, sinks)
    got, lse = run(ctx, zb, torch, cache, q, table, [length], None, kind, window=window, sinks=sinks, scale=scale)
    within(got, want, off)
    _, _, want_lse, lse_off, _ = ref.attention(cache, q[0], table, [length], None, kind, scale, window, sinks)
    within(lse, want_lse, lse_off + more, "lse")


def times(cache, pages, bits):
    cache.scales[1][pages] = np.ldexp(cache.scales[1][pages], bits)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("bits", [10, 20, 24, 30, 40, 80, 99, 120, 150])
@pytest.mark.parametrize("new,length,dim,page,window", [(160, 160, 64, 16, 0), (160, 160, 128, 16, 0), (200, 250, 128, 64, 60), (150, 150, 256, 32, 0), (5, 69, 64, 64, 0), (6, 122, 128, 16, 40)])
def test_quiet_pages_beside_loud_ones(ctx, zb, new, length, dim, page, window, bits, kind):
    """Quiet pages first, or loud ones that a window leaves behind: some rows see quiet ones alone."""
    pages = -(-length // page)
    middle = length - new // 2 - window                # where the middle row's window begins
    loud = range(1, middle // page + 1) if window else range(pages // 2, pages)

    def change(cache, pages, q):
        times(cache, pages, -70)
        times(cache, [pages[i] for i in loud], bits)
    compare(ctx, zb, new, length, 4, 2, dim, page, kind, change, window=window)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("bits", [20, 40, 70, 110])
@pytest.mark.parametrize("first", [True, False])
def test_a_loud_page_that_nobody_attends_to(ctx, zb, new, bits, first, kind):
    """Its weights are 2^-bits and less, its scale 2^(bits - 10) times the others'."""
    page, length = 32, 32 * 8

    def change(cache, pages, q):
        times(cache, pages, -60)
        loud = pages[0 if first else 3]
        times(cache, [loud], bits - 10)
        q[:] = 1.0 + 0.01 * q
        cache.codes[0][loud], cache.scales[0][loud] = -100, 0.01 * bits * 0.6931 / 64
    compare(ctx, zb, new, length, 4, 2, 64, page, kind, change, scale=1.0)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 5, 140])
@pytest.mark.parametrize("bits", [-116, -110, -60, 60, 110])
def test_all_pages_alike(ctx, zb, new, bits, kind):
    compare(ctx, zb, new, 200, 4, 2, 64, 16, kind, lambda cache, pages, q: times(cache, pages, bits))


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("page", [16, 64])
def test_scales_of_zero(ctx, zb, new, page, kind):
    """Their codes count as zeros, whatever they are, and their weights are in the sum."""
    def change(cache, pages, q):
        cache.scales[1][pages[::2]] = 0
    compare(ctx, zb, new, 260, 4, 2, 128, page, kind, change)


@pytest.mark.parametrize("new", [1, 140])
def test_every_page_its_own(ctx, zb, new):
    """Scales over the whole range of fp32, sums across pages of all of them."""
    def change(cache, pages, q):
        for i, p in enumerate(pages):
            times(cache, [p], -100 + (i * 37) % 200)
    for kind in ("bf16", "f32"):
        compare(ctx, zb, new, 400, 4, 2, 64, 16, kind, change)
