"""token_logprobs against 64 bits."""
import numpy as np
import pytest

import token_ops_reference as ref

pytestmark = pytest.mark.gpu
TYPES = ("f32", "f16", "bf16")


def torch_type(torch, t):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def run(ctx, torch, x, tokens, top, entropy=True):
    rows = x.shape[0]
    out = (None if tokens is None else torch.full((rows,), 5.0, device="cuda"), torch.full((rows,), 5.0, device="cuda") if entropy else None,
           torch.full((rows, top), -7, dtype=torch.int32, device="cuda"), torch.full((rows, top), 5.0, device="cuda"))
    torch.cuda.synchronize()
    got = ctx.token_logprobs(x, None if tokens is None else torch.from_numpy(tokens).cuda(), top=top, out=out)
    ctx.synchronize()
    assert got is out
    return [None if o is None else o.cpu().numpy() for o in out]


def near(got, want, off):
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine].astype(np.float32), equal_nan=True), (got, want)
    d = np.abs(got.astype(np.float64) - want)
    assert (d[fine] <= np.broadcast_to(off, want.shape)[fine]).all(), (float((d / off)[fine].max()), d[fine].max())


def check(got, x, tokens, top):
    x = x.double().cpu().numpy()
    given, entropy, ids, likely = ref.token_logprobs(x, tokens, top)
    log_s, h = ref.logprob_bound(x)
    # x - m is rounded, log S taken from it, the difference rounded
    with np.errstate(all="ignore"):
        if tokens is not None:
            near(got[0], given, log_s + 4 * ref.U * (1 + np.abs(np.where(np.isfinite(given), given, 0))))
        if got[1] is not None:
            near(got[1], entropy, h)
        assert np.array_equal(got[2], ids), np.argwhere(got[2] != ids)[:5]
        near(got[3], likely, log_s[:, None] + 4 * ref.U * (1 + np.abs(np.where(np.isfinite(likely), likely, 0))))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 5, 31, 32, 33, 100, 255, 257, 1000, 1024, 4099, 32000, 50257, 128256, 200001])
def test_sizes(ctx, t, vocab):
    import torch
    rng = np.random.default_rng(vocab)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for rows in (1, 3, 40) if vocab < 50000 else (1, 9):
        x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(torch_type(torch, t))
        tokens = rng.integers(0, vocab, rows).astype(np.int32)
        for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}):
            check(run(ctx, torch, x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("rows", [2, 50, 147, 149, 300, 1500, 4000])
def test_rows(ctx, rows):
    import torch
    rng = np.random.default_rng(rows)
    x = (torch.randn(rows, 2003, generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda") * 4).to(torch_type(torch, TYPES[rows % 3]))
    tokens = rng.integers(-1, 2004, rows).astype(np.int32)
    check(run(ctx, torch, x, tokens, 7), x, tokens, 7)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [40, 3000, 70000])
def test_masks(ctx, t, vocab):
    """Minus infinity at most places, at all, at the start, at the end; the type's lowest value as a mask; fewer finite logits than alternatives."""
    import torch
    d = torch_type(torch, t)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(9, vocab, generator=g, device="cuda") * 3).to(d)
    inf = float("inf")
    x[0] = -inf
    x[1, 5:] = -inf
    x[2, :vocab - 3] = -inf
    x[3, ::2] = -inf
    x[4] = torch.finfo(d).min
    x[5, 1:] = torch.finfo(d).min
    x[6, :] = -inf
    x[6, vocab // 2] = torch.finfo(d).min
    x[7] = torch.finfo(d).max
    x[8, 3] = torch.finfo(d).max
    tokens = np.array([2, 3, 0, 1, 7, 0, vocab // 2, 39, 3], np.int32)
    for top in (0, 6, 32):
        check(run(ctx, torch, x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,vocab", [(3, 70000), (260, 1819), (200, 31910)])
@pytest.mark.parametrize("share", [0.5, 0.9, 0.999])
def test_most_places_masked(ctx, t, rows, vocab, share):
    import torch
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(torch_type(torch, t))
    x[torch.rand(rows, vocab, generator=g, device="cuda") < share] = -float("inf")
    tokens = np.random.default_rng(rows).integers(0, vocab, rows).astype(np.int32)
    for top in (0, 5):
        check(run(ctx, torch, x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [33, 5000])
def test_nan_and_infinity(ctx, t, vocab):
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(8, vocab, generator=g, device="cuda").to(torch_type(torch, t))
    inf, nan = float("inf"), float("nan")
    x[0, 9] = nan
    x[1, 30] = inf
    x[2, [3, 30]] = inf
    x[3, 4], x[3, 2] = nan, inf
    x[4] = nan
    x[5] = -inf
    x[5, 7] = nan
    x[6] = -inf
    x[6, 7] = inf
    tokens = np.full(8, 7, np.int32)
    for top in (0, 4, 32):
        check(run(ctx, torch, x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [32, 700, 20000, 131072])
def test_ties(ctx, t, vocab):
    """Equal logits: the lower id first, whatever order they are met in; -0 and +0 are equal; falling and rising rows."""
    import torch
    d = torch_type(torch, t)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.zeros(8, vocab, device="cuda")
    x[0, ::2] = -0.0
    x[1] = torch.randint(0, 4, (vocab,), generator=g, device="cuda").float()
    x[2] = torch.arange(vocab, device="cuda").float() * (20.0 / vocab)
    x[3] = -x[2]
    x[4] = torch.randint(0, vocab // 8 + 1, (vocab,), generator=g, device="cuda").float() * 0.01
    x[5, vocab - 1] = 1
    x[6, [0, vocab // 2, vocab - 1]] = 3
    x[7] = (torch.arange(vocab, device="cuda") % 7).float()
    x = x.to(d)
    tokens = np.arange(8, dtype=np.int32)
    for top in (1, 3, 32):
        check(run(ctx, torch, x, tokens, top), x, tokens, top)


def test_given_tokens(ctx):
    import torch
    x = torch.randn(6, 300, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    tokens = np.array([-1, 300, 2 ** 31 - 1, -2 ** 31, 0, 299], np.int32)
    got = run(ctx, torch, x, tokens, 2)
    check(got, x, tokens, 2)
    assert got[0][0] == 0 and got[0][3] == 0 and np.isnan(got[0][1:3]).all()


def test_parts(ctx):
    """Any of the results may be left out."""
    import torch
    x = torch.randn(5, 4000, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    tokens = np.array([1, 2, 3, 4, 5], np.int32)
    for tk in (tokens, None):
        for entropy in (True, False):
            for top in (0, 9):
                check(run(ctx, torch, x, tk, top, entropy), x, tk, top)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [1000, 40000])
def test_strides_and_addresses(ctx, t, vocab):
    import torch
    room = torch.randn(7, vocab + 50, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").to(torch_type(torch, t))
    tokens = np.array([0, vocab - 1, 5, 6, 7, 8, 9], np.int32)
    for off in (0, 1, 2, 5, 8, 16):
        for n in (vocab, vocab - 3):
            x = room[:, off:off + n]
            tk = np.minimum(tokens, n - 1)
            check(run(ctx, torch, x, tk, 10), x, tk, 10)


def test_far_rows(ctx):
    import torch
    x = torch.empty(2 ** 31 + 4096, dtype=torch.float16, device="cuda").as_strided((2, 3000), (2 ** 31 + 8, 1))
    x.copy_(torch.randn(2, 3000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)))
    tokens = np.array([5, 2999], np.int32)
    check(run(ctx, torch, x, tokens, 20), x, tokens, 20)


def test_large_offsets_of_logits(ctx):
    """exp does not overflow, and small probabilities are not lost: logits around +-1000."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(8)
    for shift in (-1000.0, 1000.0):
        for scale in (0.01, 1.0, 100.0):
            x = torch.randn(4, 9000, generator=g, device="cuda") * scale + shift
            tokens = np.array([0, 1, 2, 8999], np.int32)
            check(run(ctx, torch, x, tokens, 8), x, tokens, 8)


def test_host_arrays(ctx):
    rng = np.random.default_rng(9)
    for dt in (np.float32, np.float16):
        x = rng.standard_normal((4, 1234)).astype(dt)
        tokens = [1, 5, -1, 1233]
        got = ctx.token_logprobs(x, tokens, top=4)
        import torch
        check(got, torch.from_numpy(x), np.array(tokens, np.int32), 4)
