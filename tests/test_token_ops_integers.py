"""Indices, tokens and offsets in host arrays of other types than int32: whole numbers keep their meaning, anything else is refused."""
import numpy as np
import pytest

import token_ops_reference as ref

F = np.float32


def test_others_than_whole_numbers_are_refused(zb):
    nogpu = zb.Context(None)
    x, a, w = np.ones((2, 8), F), np.ones((2, 8), np.int8), np.ones((1, 5, 8), np.int8)
    for bad in ([0.0, 1.0], [0.5, 1], [float("nan"), 0], ["0", "1"], [2 ** 70, 0]):
        for call in (lambda: nogpu.quantize_rows(x, index=bad), lambda: nogpu.token_logprobs(x, bad), lambda: nogpu.qmatmul_grouped(a, np.ones(2, F), w, np.ones((1, 5), F), bad)):
            with pytest.raises(zb.ZantError) as e:
                call()
            assert e.value.name == "InputArrayWrongType"
    for good in ([0, 1], np.array([0, 2 ** 40]), np.array([2 ** 63, 1], np.uint64), np.array([1, 0], np.int8)):
        for call in (lambda: nogpu.quantize_rows(x, index=good), lambda: nogpu.token_logprobs(x, good), lambda: nogpu.qmatmul_grouped(a, np.ones(2, F), w, np.ones((1, 5), F), good)):
            with pytest.raises(zb.ZantError) as e:
                call()
            assert e.value.name == "CudaUnavailable"
    q, s = nogpu.quantize_rows(x, index=[])
    assert q.shape == (0, 8) and s.shape == (0,)


FAR = [np.array([1, 2 ** 32 + 1, -2 ** 32, 2 ** 31, 2 ** 63 - 1, -1, 2]), np.array([1, 2 ** 32, 2 ** 64 - 1, 2 ** 63, 2], np.uint64), np.array([2 ** 32 - 1, 0, 2], np.uint32)]


@pytest.mark.gpu
@pytest.mark.parametrize("far", FAR, ids=lambda v: str(v.dtype))
def test_numbers_beyond_int32_lie_outside(ctx, far):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 40)).astype(F)
    exact = np.array([int(v) if -2 ** 31 <= int(v) < 2 ** 31 else (2 ** 31 - 1 if int(v) > 0 else -2 ** 31) for v in far])
    q, s = ctx.quantize_rows(x, index=far)
    wq, ws = ref.quantize_rows(x.astype(np.float64), exact)
    assert np.array_equal(q, wq) and np.array_equal(s, ws)
    logits = rng.standard_normal((len(far), 30)).astype(F)
    got = ctx.token_logprobs(logits, far)[0]
    want = ref.token_logprobs(logits.astype(np.float64), exact, 0)[0]
    # (30 logits: about 70 roundings of 2**-24 and the results' own, a fifth of this)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.allclose(got, want, rtol=0, atol=1e-5, equal_nan=True)


@pytest.mark.gpu
def test_offsets_beyond_int32_are_clamped(ctx):
    rng = np.random.default_rng(1)
    a, w = rng.integers(-127, 128, (9, 32), dtype=np.int8), rng.integers(-127, 128, (3, 5, 32), dtype=np.int8)
    one = np.ones(9, F), np.ones((3, 5), F)
    out = np.full((9, 5), 77, F)
    ctx.qmatmul_grouped(a, one[0], w, one[1], np.array([-2 ** 40, 2, 2 ** 33, 2 ** 40]), out=out)
    full = a.astype(np.int64) @ w.astype(np.int64).transpose(0, 2, 1)
    assert np.array_equal(out[:2], full[0][:2]) and np.array_equal(out[2:], full[1][2:])
