"""What NaN and infinities in queries and in scales of pages do to kv_cache_attention: rows that see them have NaN, also where the weight is nothing; rows that do not see them have what they would have without."""
import numpy as np
import pytest

import decode_ops_reference as ref
from test_gpu_kv_attention import run, within
from test_gpu_kv_cache import as_kind, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [5, 90])
def test_a_query_that_sees_nothing_has_zeros_whatever_it_is(ctx, zb, new, kind):
    import torch
    rng = np.random.default_rng(1)
    cache = ref.Cache(12, 2, 16, 64, rng)
    table = tables(rng, 12, 16, [new - 2, new - 2])
    table[1, :] = -1
    q = rng.standard_normal((2 * new, 4, 64))
    q[0, 1, 3] = q[3, 2, 5] = np.nan             # sees nothing (position -2); sees its own tokens
    q[1, 0, 0], q[new + 4, 1, 7] = np.inf, np.nan
    q = as_kind(torch, q, kind)
    want, off, lse, lse_off, _ = ref.attention(cache, np.where(np.isfinite(q[0]), q[0], 0), table, [new - 2, new - 2], None, kind)
    got, got_lse = run(ctx, zb, torch, cache, q, table, [new - 2, new - 2], None, kind)
    assert np.isnan(got[3, 2]).all() and np.isnan(got_lse[3, 2])
    rest = np.ones(got.shape[:2], bool)
    rest[3, 2] = False
    within(got[rest], want[rest], off[rest])
    none = np.isneginf(lse)
    assert none[:2].all() and none[new:].all() and (got[none] == 0).all() and np.isneginf(got_lse[none]).all()
    within(got_lse[rest & ~none], lse[rest & ~none], lse_off[rest & ~none], "lse")


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new,page,window", [(2, 16, 50), (2, 64, 70), (100, 16, 50), (100, 64, 70)])
def test_scales_that_are_no_numbers(ctx, zb, new, page, window, kind, kv, bad):
    """On a page that some rows see and others do not, and on one that nobody sees."""
    import torch
    rng = np.random.default_rng(2)
    length, pages = 400, -(-400 // page)
    cache = ref.Cache(pages, 2, page, 64, rng)
    table = tables(rng, pages, page, [length])
    first = length - new
    spoilt = (first - window + 1 + new // 2) // page          # the page where the window of the middle row begins
    clean = cache.copy()
    for at in (spoilt, 0):
        cache.scales[kv][table[0, at], 0] = bad
    q = as_kind(torch, rng.standard_normal((new, 4, 64)), kind)
    want, off, _, _, _ = ref.attention(clean, q[0], table, [length], None, kind, None, window, 0)
    got, _ = run(ctx, zb, torch, cache, q, table, [length], None, kind, window=window)
    nan = np.zeros(got.shape[:2], bool)
    for i in range(new):
        low = first + i - window + 1
        nan[i, :2] = low // page <= spoilt
    assert nan.any()
    assert np.array_equal(np.isnan(got).all(2), nan) and np.array_equal(np.isnan(got).any(2), nan)
    within(got[~nan], want[~nan], off[~nan])


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [2, 100])
@pytest.mark.parametrize("page", [16, 32])
def test_a_weight_of_nothing(ctx, zb, page, new, kind, bad):
    """Scores 400 below the others': the page is seen all the same."""
    import torch
    rng = np.random.default_rng(3)
    cache = ref.Cache(20, 1, page, 64, rng)
    table = tables(rng, 20, page, [300])
    cache.codes[0][:], cache.scales[0][:] = 100, 0.01
    cache.codes[0][table[0, 2]] = -100
    cache.scales[1][table[0, 2]] = bad
    q = as_kind(torch, np.full((new, 2, 64), 25.0), kind)
    got, _ = run(ctx, zb, torch, cache, q, table, [300], None, kind)
    assert np.isnan(got).all()
