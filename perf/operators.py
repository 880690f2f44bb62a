"""Workloads of the operators that language models add to the int8 path.

Kinds
  linear    a linear layer on activations that are quantized as they come: quantize_rows (one scale for each token), then
            qmatmul_scaled (int8 weights [out, in] with one scale for each output channel)
  experts   the same for a mixture of experts: quantize_rows gathers the tokens into the order of their experts, then
            qmatmul_grouped multiplies each expert's rows with that expert's weights; how many rows an expert gets is known
            on the device only
  logprobs  token_logprobs: log probabilities of given tokens, entropy of the distribution, the likeliest alternatives

`listed()` are the fixed cases, `draw(rng)` gives more of the same ranges, `prepare` makes what a program holds before the call,
`run` is one pass: in plain torch operations, or through the package where `own` is set.  `exact` states the result in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MOST_OPS = 2 * 8192 ** 3            # of the largest listed product
MOST_LOGITS = 4096 * 65536 * 2      # bytes of the largest listed logits


def listed():
    return [
        # one sequence, one token at a time: latency
        dict(name="linear_1x4096x4096", kind="linear", rows=1, k=4096, n=4096, x="bf16", y="bf16", bias=False),
        # a decoding batch, the wide layer of a block: the weights' bytes
        dict(name="linear_48x4096x12288", kind="linear", rows=48, k=4096, n=12288, x="bf16", y="bf16", bias=False),
        # sizes that are multiples of nothing; rows that start at odd addresses
        dict(name="linear_257x4095x5001", kind="linear", rows=257, k=4095, n=5001, x="f16", y="f16", bias=True),
        # a prompt of ordinary length, float32 on both sides
        dict(name="linear_2048x2048x8192_f32", kind="linear", rows=2048, k=2048, n=8192, x="f32", y="f32", bias=True),
        # a batch of long prompts
        dict(name="linear_8192x8192x8192", kind="linear", rows=8192, k=8192, n=8192, x="bf16", y="bf16", bias=False),
        # decoding with many small experts: most get one or two rows, some none
        dict(name="experts_16of64_2048x1536", kind="experts", tokens=16, top=6, experts=64, k=2048, n=1536, x="bf16", y="bf16", bias=False, spare=0),
        # a prompt over experts of unequal popularity
        dict(name="experts_4096of32_2048x2816", kind="experts", tokens=4096, top=4, experts=32, k=2048, n=2816, x="bf16", y="bf16", bias=False, spare=0),
        # a padded batch (rows behind the last expert stay as they are) of odd sizes
        dict(name="experts_333of7_1000x1503", kind="experts", tokens=333, top=2, experts=7, k=1000, n=1503, x="f32", y="f32", bias=True, spare=30),
        # the next token of one sequence
        dict(name="logprobs_1x32000", kind="logprobs", rows=1, vocab=32000, top=5, x="f16", masked=0.0),
        # a decoding batch with a mask from a grammar
        dict(name="logprobs_64x128000_top20", kind="logprobs", rows=64, vocab=128000, top=20, x="bf16", masked=0.3),
        # scoring a text: no alternatives, odd vocabulary
        dict(name="logprobs_1000x50001_f32", kind="logprobs", rows=1000, vocab=50001, top=0, x="f32", masked=0.0),
        # scoring a batch of long texts, with the likeliest token for comparison
        dict(name="logprobs_4096x65536_top1", kind="logprobs", rows=4096, vocab=65536, top=1, x="bf16", masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """Three of four sizes are what layers have (multiples of 64), the fourth is any."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < 0.25 else max(64, v // 64 * 64)


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "logprobs"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    y = rng.choice([x, x, "f32"])
    if kind == "linear":
        k, n = _size(rng, 512, 12288), _size(rng, 512, 12288)
        rows = _log_int(rng, 1, max(1, min(8192, MOST_OPS // (4 * k * n))))
        return dict(kind=kind, rows=rows, k=k, n=n, x=x, y=y, bias=rng.random() < 0.3)
    if kind == "experts":
        k, n = _size(rng, 256, 4096), _size(rng, 256, 4096)
        experts = _log_int(rng, 4, 128)
        top = rng.randint(1, min(8, experts))
        return dict(kind=kind, tokens=_log_int(rng, 1, 4096), top=top, experts=experts, k=k, n=n, x=x, y=y, bias=rng.random() < 0.3, spare=rng.choice([0, 0, rng.randint(1, 40)]))
    vocab = _log_int(rng, 1000, 160000)
    rows = _log_int(rng, 1, max(1, min(4096, MOST_LOGITS // (vocab * BYTES[x]))))
    return dict(kind=kind, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]), x=x, masked=rng.choice([0.0, 0.0, 0.3, 0.9]))


def _activations(g, rows, k, x):
    """Roughly normal, with a few channels that are much larger than the others, as hidden states are."""
    v = torch.randn(rows, k, generator=g, device="cuda")
    loud = 1 + 15 * (torch.rand(k, generator=g, device="cuda") < 0.005).float()
    return (v * loud * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))).to(TORCH[x])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, dev = case, "cuda"
    if c["kind"] == "logprobs":
        logits = torch.randn(c["rows"], c["vocab"], generator=g, device=dev) * 3
        if c["masked"]:
            logits.masked_fill_(torch.rand(c["rows"], c["vocab"], generator=g, device=dev) < c["masked"], -math.inf)
        logits = logits.to(TORCH[c["x"]])
        tokens = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=dev, dtype=torch.int32)
        out = (torch.empty(c["rows"], device=dev), torch.empty(c["rows"], device=dev),
               torch.empty(c["rows"], c["top"], dtype=torch.int32, device=dev), torch.empty(c["rows"], c["top"], device=dev))
        return dict(case=c, logits=logits, tokens=tokens, out=out)
    k, n = c["k"], c["n"]
    experts = c.get("experts", 1)
    w = torch.randint(-127, 128, (experts, n, k), generator=g, device=dev, dtype=torch.int8)
    w_scale = (0.5 + torch.rand(experts, n, generator=g, device=dev)) / (73.0 * math.sqrt(k))
    bias = torch.randn(experts, n, generator=g, device=dev) if c["bias"] else None
    room = -(-k // 16) * 16                      # codes in rows of whole 16-byte units
    if c["kind"] == "linear":
        rows = c["rows"]
        return dict(case=c, x=_activations(g, rows, k, c["x"]), w=w[0], w_scale=w_scale[0], bias=None if bias is None else bias[0],
                    q=torch.zeros(rows, room, dtype=torch.int8, device=dev)[:, :k], s=torch.empty(rows, device=dev),
                    out=torch.empty(rows, n, dtype=TORCH[c["y"]], device=dev))
    # each token goes to `top` different experts; popular ones get several times the rows of others
    logits = torch.randn(c["tokens"], experts, generator=g, device=dev) + torch.randn(experts, generator=g, device=dev)
    chosen = logits.argsort(dim=1, descending=True)[:, :c["top"]].reshape(-1)
    order = torch.argsort(chosen, stable=True)
    index = (order // c["top"]).to(torch.int32)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=dev)
    offsets[1:] = torch.bincount(chosen, minlength=experts).cumsum(0)
    rows = c["tokens"] * c["top"] + c["spare"]
    index = torch.cat([index, torch.full((c["spare"],), -1, dtype=torch.int32, device=dev)])
    return dict(case=c, x=_activations(g, c["tokens"], k, c["x"]), index=index, offsets=offsets, w=w, w_scale=w_scale, bias=bias,
                q=torch.zeros(rows, room, dtype=torch.int8, device=dev)[:, :k], s=torch.empty(rows, device=dev),
                out=torch.zeros(rows, n, dtype=TORCH[c["y"]], device=dev))


# --------------------------------------------------------------------------------------------- through the package
_held = {}


def _context():
    """The package and a context on torch's current stream, kept by the program."""
    if not _held:
        import __graft_entry__ as entry
        _held["zb"] = entry.load_package()
        _held["ctx"] = _held["zb"].Context(0)
        _held["ctx"].set_stream(torch.cuda.current_stream().cuda_stream)
    return _held["ctx"]


def _run_own(s):
    ctx = _context()
    kind = s["case"]["kind"]
    if kind == "linear":
        ctx.quantize_rows(s["x"], out=s["q"], out_scale=s["s"])
        return ctx.qmatmul_scaled(s["q"], s["s"], s["w"], s["w_scale"], bias=s["bias"], out=s["out"])
    if kind == "experts":
        ctx.quantize_rows(s["x"], index=s["index"], out=s["q"], out_scale=s["s"])
        return ctx.qmatmul_grouped(s["q"], s["s"], s["w"], s["w_scale"], s["offsets"], bias=s["bias"], out=s["out"])
    return ctx.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"], out=s["out"])


# --------------------------------------------------------------------------------------------- plain form
def _plain_codes(x):
    x = x.float()
    scale = (x.abs().amax(dim=1).double() / 127).float()
    # next to a border between two codes a quotient of 32 bits may land on the wrong side
    q = torch.round(x.double() / scale.double()[:, None]).clamp(-127, 127)
    return torch.where(scale[:, None] > 0, q, 0.0).float(), scale


def _plain_product(q, scale, w, w_scale, bias):
    y = (q @ w.float().T) * scale[:, None] * w_scale
    return y if bias is None else y + bias


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "linear":
        q, scale = _plain_codes(s["x"])
        return _plain_product(q, scale, s["w"], s["w_scale"], s["bias"]).to(TORCH[c["y"]])
    if c["kind"] == "experts":
        ends = s["offsets"].tolist()
        q, scale = _plain_codes(s["x"].index_select(0, s["index"][:ends[-1]]))
        y = torch.zeros_like(s["out"])
        for e in range(c["experts"]):
            b, f = ends[e], ends[e + 1]
            if f > b:
                y[b:f] = _plain_product(q[b:f], scale[b:f], s["w"][e], s["w_scale"][e], None if s["bias"] is None else s["bias"][e]).to(y.dtype)
        return y
    x = s["logits"].float()
    d = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    logp = d - torch.log(total)
    entropy = torch.log(total[:, 0]) - torch.where(e > 0, e * d, 0.0).sum(dim=1) / total[:, 0]
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]] if c["top"] else torch.zeros(c["rows"], 0, dtype=torch.int64, device=x.device)
    return logp.gather(1, s["tokens"].long()[:, None])[:, 0], entropy, ids.to(torch.int32), logp.gather(1, ids)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    c = case
    if c["kind"] == "logprobs":
        cells = c["rows"] * c["vocab"]
        return {"bytes": cells * BYTES[c["x"]] + c["rows"] * (12 + 8 * c["top"]), "flops": 6 * cells}
    if c["kind"] == "linear":
        rows, groups, x_rows = c["rows"], 1, c["rows"]
    else:
        # experts that get a row at all, as if all were equally popular
        rows, x_rows = c["tokens"] * c["top"], c["tokens"]
        groups = c["experts"] * (1 - (1 - c["top"] / c["experts"]) ** c["tokens"])
    moved = x_rows * c["k"] * BYTES[c["x"]] + groups * c["n"] * (c["k"] + 4 + (4 if c["bias"] else 0)) + rows * c["n"] * BYTES[c["y"]]
    return {"bytes": moved, "flops": 2 * rows * c["k"] * c["n"]}


# --------------------------------------------------------------------------------------------- 64 bits
def _exact_rows(x, w, w_scale, bias):
    x = x.to(torch.float64)
    top = x.abs().max(dim=1).values
    scale = (top / 127.0).to(torch.float32).to(torch.float64)       # the scale is a number of 32 bits
    codes = torch.round(x / torch.where(scale == 0, torch.ones_like(scale), scale).unsqueeze(1))
    codes.clamp_(-127.0, 127.0).mul_((scale != 0).to(torch.float64).unsqueeze(1))
    sums = torch.mm(codes, w.to(torch.float64).t())                 # whole numbers below 2**53
    sums.mul_(scale.unsqueeze(1)).mul_(w_scale.to(torch.float64).unsqueeze(0))
    return sums if bias is None else sums.add_(bias.to(torch.float64).unsqueeze(0))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _exact_rows(s["x"], s["w"], s["w_scale"], s["bias"])
    if case["kind"] == "experts":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        off = np.asarray(s["offsets"].cpu())
        for e in np.flatnonzero(np.diff(off)):
            lo, hi = int(off[e]), int(off[e + 1])
            out[lo:hi] = _exact_rows(s["x"][s["index"][lo:hi].long()], s["w"][e], s["w_scale"][e], None if s["bias"] is None else s["bias"][e])
        return out
    given, spread, likely = [], [], []
    top = case["top"]
    for at in range(0, case["rows"], 256):          # a part at a time: 64 bits of all would be several times the card's share
        x = s["logits"][at:at + 256].to(torch.float64)
        logs = x - torch.logsumexp(x, dim=1).unsqueeze(1)
        p = torch.exp(logs)
        given.append(torch.take_along_dim(logs, s["tokens"][at:at + 256].long().unsqueeze(1), 1).squeeze(1))
        spread.append(torch.where(p == 0, torch.zeros_like(p), -p * logs).sum(1))
        likely.append(torch.topk(logs, top, dim=1).values if top else logs[:, :0])
    return torch.cat(given), torch.cat(spread), None, torch.cat(likely)
