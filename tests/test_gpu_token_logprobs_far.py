"""token_logprobs of rows whose maximum is far from zero: the distance of a logit from the maximum counts, not its size."""
import numpy as np
import pytest

import token_ops_reference as ref
from test_gpu_token_logprobs import near, run, torch_type

pytestmark = pytest.mark.gpu
FAR = [-3e38, -1e30, -2e25, -1e20, -2e12, -1e10, -1e9, -3e7, -2.0 ** 22, -4194303.0, -1e5, 1e5, 4194303.0, 2.0 ** 22, 5e6, 3e7, 1e9, 3e10, 2e12, 1e20, 5e30, 1e37, 3e38]


def check(got, x, tokens, top):
    """As the check of ordinary rows, but for log p below the lowest fp32 number: at or beyond 2**128 - 2**103, half a step behind the largest number
    2**128 - 2**104, to the nearest is infinity."""
    x = x.double().cpu().numpy()
    given, entropy, ids, likely = ref.token_logprobs(x, tokens, top)
    given, likely = (np.where(v <= -(2.0 ** 128 - 2.0 ** 103), -np.inf, v) for v in (given, likely))
    log_s, h = ref.logprob_bound(x)
    with np.errstate(all="ignore"):
        near(got[0], given, log_s + 4 * ref.U * (1 + np.abs(np.where(np.isfinite(given), given, 0))))
        near(got[1], entropy, h)
        assert np.array_equal(got[2], ids)
        near(got[3], likely, log_s[:, None] + 4 * ref.U * (1 + np.abs(np.where(np.isfinite(likely), likely, 0))))


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [33, 5000, 70000])
def test_maxima_far_from_zero(ctx, t, vocab):
    """Equal logits throughout (a mask of some low number that leaves nothing), neighbours of the maximum, one logit among masked and among ordinary ones."""
    import torch
    d = torch_type(torch, t)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows = []
    far = FAR if t != "f16" else [-65504.0, -65440.0, -65280.0, -60000.0, -3e4, 3e4, 60000.0, 65504.0]
    for m in far:
        at = int(torch.randint(0, vocab, (1,), generator=g, device="cuda"))
        equal = torch.full((vocab,), m, device="cuda")
        near = (equal.double() * (1 + torch.finfo(d).eps * torch.randint(-3, 1 if m > 0 else 4, (vocab,), generator=g, device="cuda"))).float()
        alone = torch.full((vocab,), -float("inf"), device="cuda")
        alone[at] = m
        among = torch.randn(vocab, generator=g, device="cuda") * 3
        among[at] = m
        above = equal.clone() if m < 0 else torch.full((vocab,), -m, device="cuda")
        above[at] = abs(m) if m > 0 else m * 0.5
        rows += [equal, near, alone, among, above]
    x = torch.stack(rows).to(d)
    assert torch.isfinite(x.float().amax(dim=1)).all()
    tokens = np.random.default_rng(vocab).integers(0, vocab, len(rows)).astype(np.int32)
    for top in (0, 4, 32):
        check(run(ctx, torch, x, tokens, top), x, tokens, top)
        few = slice(len(rows) // 2 - 3, len(rows) // 2 + 3)          # (few rows: several CTAs a row)
        check(run(ctx, torch, x[few], tokens[few], top), x[few], tokens[few], top)
