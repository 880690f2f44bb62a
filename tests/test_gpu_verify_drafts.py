"""verify_drafts against its plain form: whole numbers, equal in every place."""
import numpy as np
import pytest

import decode_ops_reference as ref
from test_gpu_kv_cache import as_kind, ints

pytestmark = pytest.mark.gpu


def softmax(x):
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def both(ctx, torch, target, drafted, tokens, accept, sample, offsets, stride=0):
    seqs = len(sample)
    p, q = target[1], None if drafted is None else drafted[1]
    if stride:
        wide = lambda t: torch.zeros(t.shape[0], t.shape[1] + stride, dtype=t.dtype, device="cuda")[:, 1:1 + t.shape[1]].copy_(t)  # noqa: E731
        p, q = wide(p), None if q is None else wide(q)
    f = lambda v: torch.from_numpy(np.asarray(v, np.float32)).cuda()  # noqa: E731
    dk, do = ints(torch, tokens, offsets)
    out = tuple(torch.full((seqs,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    ctx.verify_drafts(p, q, dk, f(accept), f(sample), offsets=do, out=out)
    ctx.synchronize()
    want = ref.verify(target[0], None if drafted is None else drafted[0], tokens, np.asarray(accept, np.float32), np.asarray(sample, np.float32), offsets)
    got = [o.cpu().numpy() for o in out]
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    return got


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seqs,drafts,vocab,drafted,ragged,stride", [
    (1, 1, 1, True, False, 0), (1, 0, 7, True, False, 0), (2, 1, 2, True, False, 0), (3, 4, 31, True, False, 0), (1, 40, 50, True, False, 0), (5, 3, 1000, False, False, 0),
    (4, 5, 4097, True, True, 0), (7, 6, 5003, False, True, 2), (2, 3, 32000, True, False, 0), (40, 2, 8200, True, True, 3), (300, 1, 700, True, False, 0), (1, 5, 128001, True, False, 0)])
def test_drafts(ctx, kind, seqs, drafts, vocab, drafted, ragged, stride):
    import torch
    rng = np.random.default_rng(seqs * 100 + vocab)
    counts = rng.integers(0, drafts + 1, seqs) if ragged else np.full(seqs, drafts)
    n = int(counts.sum())
    offsets = np.concatenate([[0], np.cumsum(counts)]) if ragged else None
    logits = rng.standard_normal((n + seqs, vocab)) * 2
    rows = np.arange(n) + np.repeat(np.arange(seqs), counts)
    near = logits[rows] + rng.standard_normal((n, vocab)) * 0.3
    target = as_kind(torch, softmax(logits), kind)
    small = as_kind(torch, softmax(near) if n else np.zeros((0, vocab)), kind) if drafted else None
    tokens = np.array([rng.choice(vocab, p=r) for r in (softmax(near) if n else [])], np.int64)
    for _ in range(3):
        both(ctx, torch, target, small, tokens, rng.random(n), rng.random(seqs), offsets, stride)


def test_padding_and_tokens_outside(ctx):
    """A negative token ends a sequence's drafts (the row behind them is the target's own), one beyond the vocabulary does not stand."""
    import torch
    rng = np.random.default_rng(0)
    target, drafted = (as_kind(torch, softmax(rng.standard_normal((n, 40))), "f32") for n in (16 + 4, 16))
    tokens = np.array([3, -1, 5, 6, 40, 1, 2, 3, -1, -1, -1, -1, 7, 8, 9, 2 ** 31 - 1])
    for none in (False, True):
        got = both(ctx, torch, target, None if none else drafted, tokens, np.zeros(16), rng.random(4), None)
        assert list(got[0]) == [1, 0, 0, 3]


def test_ends(ctx):
    """Numbers at the ends, equal rows, rows of nothing, probabilities that are none."""
    import torch
    p = np.zeros((8, 9))
    p[:, 2], p[:, 5] = 0.25, 0.75
    p[4] = 0
    p[6, 3], p[6, 4], p[6, 0] = np.nan, np.inf, -1.0
    q = np.zeros((4, 9))
    q[0], q[1], q[2] = p[0], p[2], 1.0
    q[3, 5] = 1.0
    tokens = np.array([2, 5, 2, 5])
    t, d = as_kind(torch, p, "f32"), as_kind(torch, q, "f32")
    for accept in (0.0, 0.5, 0.9999999, 1.0):
        for sample in (0.0, 0.25, 0.2500001, 0.9999999, 1.0):
            both(ctx, torch, t, d, tokens, [accept] * 4, [sample] * 4, None)
            both(ctx, torch, t, None, tokens, [accept] * 4, [sample] * 4, None)


def test_borders_of_a_flat_distribution(ctx):
    """Every token's border in a long running sum: u * total next to a whole number of equal steps (exact in fp64, far from it in fp32)."""
    import torch
    vocab, seqs = 100003, 64
    rng = np.random.default_rng(1)
    p = np.full((seqs, vocab), np.float32(1 / 131072), np.float64)
    want = rng.integers(0, vocab, seqs)
    u = np.nextafter(((want + 0.5) / vocab).astype(np.float32), np.float32(0))
    got = both(ctx, torch, as_kind(torch, p, "f32"), None, np.zeros(0, np.int64), [], u, None)
    assert np.abs(got[1] - want).max() <= 1


def test_host_arrays(ctx):
    rng = np.random.default_rng(2)
    p, q = softmax(rng.standard_normal((9, 50))).astype(np.float32), softmax(rng.standard_normal((6, 50))).astype(np.float32)
    tokens, a, s = rng.integers(0, 50, 6), rng.random(6).astype(np.float32), rng.random(3).astype(np.float32)
    got = ctx.verify_drafts(p, q, tokens, a, s)
    want = ref.verify(p.astype(np.float64), q.astype(np.float64), tokens, a, s, None)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
