"""verify_drafts where probabilities are NaN, negative or infinite: each counts as 0 in what is left of a row, the target's and the drafted ones alike."""
import numpy as np
import pytest

from test_gpu_kv_cache import as_kind, ints

pytestmark = pytest.mark.gpu


def following(p, q, u):
    """The token behind a draft that does not stand, with q of nothing behind one that does."""
    clean = lambda x: np.where((x > 0) & np.isfinite(x), x, 0.0)  # noqa: E731
    r = np.maximum(clean(p) - clean(q), 0.0)
    if r.sum() == 0:
        r = clean(p)
    if r.sum() == 0:
        return -1
    above = np.flatnonzero((np.cumsum(r) > u * np.cumsum(r)[-1]) & (r > 0))
    return above[0] if len(above) else np.flatnonzero(r > 0)[-1]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [9, 700, 20001])
@pytest.mark.parametrize("where", ["target", "drafted", "both"])
def test_probabilities_that_are_none(ctx, kind, vocab, where):
    import torch
    rng = np.random.default_rng(vocab)
    seqs, bad = 40, np.array([np.nan, np.inf, -np.inf, -0.25, -1e-30, 0.0])
    # multiples of 2^-7 below 2: sums of them are exact, and so is each border (16 bits hold them, too)
    p, q = (rng.integers(0, 256, (n, vocab)) / 128.0 for n in (2 * seqs, seqs))
    for x in {"target": (p,), "drafted": (q,), "both": (p, q)}[where]:
        hit = rng.random(x.shape) < 0.3
        x[hit] = rng.choice(bad, hit.sum())
    p[::2, 0] = 0.0                                   # the draft, token 0, stands against a negative number alone
    if where != "target":
        q[0], q[1] = np.nan, -1.0                     # nothing is taken away
        q[2] = np.inf
    p[6], q[3] = 0.25, 2.0                            # nothing is left: the row itself
    sample = (rng.integers(0, 64, seqs) / 64.0).astype(np.float32)
    t, d = as_kind(torch, p, kind), as_kind(torch, q, kind)
    out = tuple(torch.full((seqs,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    f = lambda v: torch.from_numpy(np.asarray(v, np.float32)).cuda()  # noqa: E731
    ctx.verify_drafts(t[1], d[1], ints(torch, np.zeros(seqs))[0], f(np.full(seqs, 0.5)), f(sample), out=out)
    ctx.synchronize()
    stands = 0.5 * d[0][:, 0] < t[0][::2, 0]
    assert np.array_equal(out[0].cpu().numpy(), stands)
    want = [following(t[0][2 * s + 1], np.zeros(vocab), float(sample[s])) if stands[s] else following(t[0][2 * s], d[0][s], float(sample[s])) for s in range(seqs)]
    assert np.array_equal(out[1].cpu().numpy(), want)
