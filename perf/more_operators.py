"""Workloads of the operators that a decoder's int8 cache adds, and of the check of drafted tokens.

Kinds
  attend    kv_cache_attention: new tokens attend to a paged cache of int8 codes with one scale for each page and head; a sliding
            window and first tokens that stay visible (sinks) where the case has them
  append    kv_cache_write quantizes the keys and values of new tokens into the cache's pages (the scale of a page that was begun
            before grows and its codes follow), then kv_cache_read brings back the pages that were written to
  verify    verify_drafts: which of a sequence's drafted tokens stand against the target's probabilities, and the token behind them

`listed()` are the fixed cases, `draw(rng)` gives more of the same ranges, `prepare` makes what a program holds before the call,
`run` is one pass: in plain torch operations, or through the package where `own` is set.  `exact` states the result in 64 bits.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
GOLDEN = 0.6180339887498949
MOST_PAIRS = 40 * 8192 * 4096 * 128        # (query, key) pairs of all heads times the head's size, of the largest listed prompt
MOST_CACHE = 1 << 29                       # bytes of codes


def listed():
    return [
        # one sequence, one token at a time, a short context: latency
        dict(name="attend_1x1_of_700", kind="attend", seqs=1, new=1, ragged=False, context=699, heads=40, kv_heads=8, dim=128, page=32, x="bf16", window=0, sinks=0),
        # a decoding batch, contexts of different lengths
        dict(name="attend_64x1_of_4096", kind="attend", seqs=64, new=1, ragged=False, context=4096, heads=40, kv_heads=8, dim=128, page=32, x="bf16", window=0, sinks=0),
        # one sequence over a very long document
        dict(name="attend_1x1_of_131072", kind="attend", seqs=1, new=1, ragged=False, context=131071, heads=64, kv_heads=8, dim=128, page=128, x="bf16", window=0, sinks=0),
        # drafted tokens of a batch, a window with sinks, pages that are smaller than any tile
        dict(name="attend_24x5_window_1024", kind="attend", seqs=24, new=5, ragged=False, context=3000, heads=16, kv_heads=4, dim=64, page=16, x="f16", window=1024, sinks=4),
        # a long prompt
        dict(name="attend_1x8192_prompt", kind="attend", seqs=1, new=8192, ragged=False, context=0, heads=40, kv_heads=8, dim=128, page=64, x="bf16", window=0, sinks=0),
        # parts of prompts of uneven lengths behind what is cached already, a window with sinks, odd head size, every head its own keys
        dict(name="attend_5x500_behind_9000", kind="attend", seqs=5, new=500, ragged=True, context=9000, heads=12, kv_heads=12, dim=96, page=64, x="f16", window=2000, sinks=8),
        # float32 tensors, a few tokens each
        dict(name="attend_7x3_of_1000_f32", kind="attend", seqs=7, new=3, ragged=True, context=1000, heads=8, kv_heads=2, dim=80, page=16, x="f32", window=0, sinks=0),
        # the decoding batch's tokens go into the cache
        dict(name="append_64x1", kind="append", seqs=64, new=1, ragged=False, context=4096, kv_heads=8, dim=128, page=32, x="bf16"),
        # a long prompt goes into the cache
        dict(name="append_1x8192", kind="append", seqs=1, new=8192, ragged=False, context=0, kv_heads=8, dim=128, page=64, x="bf16"),
        # uneven parts behind pages that were begun before, float32
        dict(name="append_9x100_f32", kind="append", seqs=9, new=100, ragged=True, context=333, kv_heads=3, dim=80, page=16, x="f32"),
        # a few sequences with three drafted tokens each
        dict(name="verify_4x3_of_32000", kind="verify", seqs=4, drafts=3, ragged=False, vocab=32000, x="f32", drafted=True),
        # a batch with uneven numbers of drafted tokens, odd vocabulary
        dict(name="verify_64x5_of_128001", kind="verify", seqs=64, drafts=5, ragged=True, vocab=128001, x="f32", drafted=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "verify"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "verify":
        vocab = _log_int(rng, 1000, 160000)
        drafts = rng.randint(1, 8)
        seqs = _log_int(rng, 1, max(1, min(128, (1 << 28) // (vocab * BYTES[x] * (2 * drafts + 1)))))
        return dict(kind=kind, seqs=seqs, drafts=drafts, ragged=rng.random() < 0.5, vocab=vocab, x=x, drafted=rng.random() < 0.8)
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12])
    if kind == "append":
        new = _log_int(rng, 1, 4096)
        seqs = _log_int(rng, 1, max(1, min(128, 65536 * 8 // (kv_heads * new * 8))))
        return dict(kind=kind, seqs=seqs, new=new, ragged=rng.random() < 0.5, context=rng.choice([0, _log_int(rng, 1, 4096)]), kv_heads=kv_heads, dim=dim, page=page, x=x)
    group = rng.choice([1, 2, 4, 5, 7, 8])
    window = rng.choice([0, 0, 128, 1000, 4096])
    if x != "f32" and rng.random() < 0.4:                 # prompts
        new, context = _log_int(rng, 100, 4096), rng.choice([0, _log_int(rng, 16, 8192)])
        while kv_heads * group * dim * new * (context + new) > MOST_PAIRS:
            new, context = new // 2 + 1, context // 2
        pairs = kv_heads * group * dim * new * (context + new)
        seqs = _log_int(rng, 1, max(1, min(8, MOST_PAIRS // (2 * pairs))))
    else:
        new, context = rng.choice([1, 1, 1, 2, 4, 7]), _log_int(rng, 16, 65536)
        seqs = _log_int(rng, 1, max(1, min(128, MOST_CACHE // (4 * kv_heads * dim * (context + new)))))
        if x == "f32":
            context = min(context, 4096)
    return dict(kind=kind, seqs=seqs, new=new, ragged=rng.random() < 0.4, context=context, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, x=x,
                window=window, sinks=rng.choice([0, 4]) if window else 0)


def _spread(i, shift):
    """Numbers between 0 and 1, as far from one another as numbers can be."""
    return ((i + 1) * GOLDEN + shift) % 1.0


def _counts(case):
    """(new tokens, tokens in the cache with them) of each sequence."""
    new = [case["new"] if not case["ragged"] else max(1, round(2 * case["new"] * _spread(i, 0.3))) for i in range(case["seqs"])]
    if case["seqs"] == 1:
        return [case["new"]], [case["context"] + case["new"]]
    return new, [n + round(case["context"] * (0.5 + _spread(i, 0.0))) for i, n in enumerate(new)]


def _draft_counts(case):
    """Drafted tokens of each sequence; some have none in an uneven batch."""
    n = case["drafts"]
    return [n if not case["ragged"] else int(_spread(i, 0.3) * (n + 1)) for i in range(case["seqs"])]


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, dev, dt = case, "cuda", TORCH[case["x"]]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if c["kind"] == "verify":
        counts = _draft_counts(c)
        starts, n, seqs, vocab = _starts(counts), sum(counts), c["seqs"], c["vocab"]
        logits = normal(n + seqs, vocab) * 3
        rows = torch.cat([torch.arange(starts[s] + s, starts[s + 1] + s, device=dev) for s in range(seqs)])      # the target's row of each drafted token
        near = logits[rows] + 0.7 * normal(n, vocab)                      # a smaller model that nearly agrees
        drafted = torch.softmax(near, 1).to(dt)
        tokens = (near - torch.log(-torch.log(torch.rand(n, vocab, generator=g, device=dev)))).argmax(1).to(torch.int32) if n else ints([])
        return dict(case=c, target=torch.softmax(logits, 1).to(dt), drafted=drafted if c["drafted"] else None, tokens=tokens, offsets=ints(starts), starts=starts,
                    accept=torch.rand(n, generator=g, device=dev), sample=torch.rand(seqs, generator=g, device=dev),
                    out=(torch.empty(seqs, dtype=torch.int32, device=dev), torch.empty(seqs, dtype=torch.int32, device=dev)))
    new, lengths = _counts(c)
    seqs, heads, page, dim = c["seqs"], c["kv_heads"], c["page"], c["dim"]
    wide = [-(-n // page) for n in lengths]
    pages = sum(wide) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((seqs, max(wide)), -1, dtype=torch.int32, device=dev)
    for s, at in enumerate(_starts(wide)[:-1]):
        table[s, :wide[s]] = order[at:at + wide[s]]
    parts = dict(k=(normal(pages, heads, page, dim) * 35).round_().clamp_(-127, 127).to(torch.int8), k_scale=(0.6 + 0.8 * torch.rand(pages, heads, generator=g, device=dev)) / 35,
                 v=(normal(pages, heads, page, dim) * 35).round_().clamp_(-127, 127).to(torch.int8), v_scale=(0.6 + 0.8 * torch.rand(pages, heads, generator=g, device=dev)) / 35)
    rows = sum(new)
    s = dict(case=c, **parts, table=table, lengths=ints(lengths), host_lengths=lengths, starts=_starts(new), offsets=ints(_starts(new)) if c["ragged"] else None)
    if c["kind"] == "attend":
        s |= dict(q=(1.5 * normal(rows, c["heads"] * dim)).to(dt), out=torch.empty(rows, c["heads"] * dim, dtype=dt, device=dev))
        return s
    # keys and values of the new tokens come from one matrix of a layer's projections
    both = (normal(rows, 2 * heads * dim) * torch.exp(0.3 * normal(rows, 1))).to(dt)
    back = [n - (n - m) // page * page for n, m in zip(lengths, new)]        # tokens of the pages that are written to
    s |= dict(new_k=both[:, :heads * dim], new_v=both[:, heads * dim:], back_starts=_starts(back), back_offsets=ints(_starts(back)),
              out=(torch.empty(sum(back), heads * dim, dtype=dt, device=dev), torch.empty(sum(back), heads * dim, dtype=dt, device=dev)))
    return s


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
    ctx, c = _context(), s["case"]
    if c["kind"] == "verify":
        return ctx.verify_drafts(s["target"], s["drafted"], s["tokens"], s["accept"], s["sample"], offsets=s["offsets"], out=s["out"])
    if "cache" not in s:
        s["cache"] = _held["zb"].KvCache(s["k"], s["k_scale"], s["v"], s["v_scale"])
    if c["kind"] == "attend":
        return ctx.kv_cache_attention(s["cache"], s["q"], s["table"], s["lengths"], offsets=s["offsets"], window=c["window"], sinks=c["sinks"], out=s["out"])
    ctx.kv_cache_write(s["cache"], s["new_k"], s["new_v"], s["table"], s["lengths"], offsets=s["offsets"])
    k, v = ctx.kv_cache_read(s["cache"], s["table"], s["lengths"], offsets=s["back_offsets"], out=s["out"])
    return k, v, s["k_scale"], s["v_scale"]


# --------------------------------------------------------------------------------------------- plain form
def _plain_tokens(codes, scale, pages):
    """[heads, tokens, dim] of a sequence's pages."""
    x = codes[pages].float() * scale[pages][:, :, None, None]
    return x.transpose(0, 1).reshape(codes.shape[1], -1, codes.shape[3])


def _plain_attend(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group = heads // kv_heads
    for i, n in enumerate(s["host_lengths"]):
        b, e = s["starts"][i], s["starts"][i + 1]
        first = n - (e - b)
        low = 0
        if c["window"]:
            low = max(0, first - c["window"] + 1) // page * page               # pages before it hold sinks at most
        low = 0 if low <= c["sinks"] else low
        pages = s["table"][i, low // page:-(-n // page)].long()
        at = torch.arange(low, n, device="cuda")
        if low and c["sinks"]:
            ahead = -(-c["sinks"] // page)
            pages = torch.cat([s["table"][i, :ahead].long(), pages])
            at = torch.cat([torch.arange(0, ahead * page, device="cuda"), at])
            drop = at[:ahead * page] >= min(c["sinks"], low)
            at[:ahead * page][drop] = n                                     # seen among the others, or by no one
        k = _plain_tokens(s["k"], s["k_scale"], pages)[:, :len(at)]
        v = _plain_tokens(s["v"], s["v_scale"], pages)[:, :len(at)]
        q = s["q"][b:e].float().view(e - b, kv_heads, group, dim)
        step = max(1, (1 << 27) // (group * len(at)))
        for r in range(0, e - b, step):
            rows = q[r:r + step]
            pos = torch.arange(first + r, first + r + len(rows), device="cuda")[:, None]
            seen = at <= pos
            if c["window"]:
                seen &= (at > pos - c["window"]) | (at < c["sinks"])
            for h in range(kv_heads):
                x = (rows[:, h].reshape(-1, dim) @ k[h].T) * (1.0 / math.sqrt(dim))
                x = x.view(len(rows), group, -1).masked_fill_(~seen[:, None], -math.inf)
                x = torch.exp(x.sub_(x.amax(-1, keepdim=True)))
                y = (x.view(-1, len(at)) @ v[h]).view(len(rows), group, dim) / x.sum(-1, keepdim=True)
                s["out"][b + r:b + r + len(rows), h * group * dim:(h + 1) * group * dim] = y.reshape(len(rows), -1).to(s["out"].dtype)
    return s["out"]


def _plain_append(s):
    c = s["case"]
    heads, dim, page = c["kv_heads"], c["dim"], c["page"]
    for x, codes, scales in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
        for i, n in enumerate(s["host_lengths"]):
            b, e = s["starts"][i], s["starts"][i + 1]
            if e == b:
                continue
            first = n - (e - b)
            p0, p1 = first // page, -(-n // page)
            pages = s["table"][i, p0:p1].long()
            pad = (first - p0 * page, p1 * page - n)
            new = torch.nn.functional.pad(x[b:e].float(), (0, 0) + pad).view(p1 - p0, page, heads, dim).transpose(1, 2)
            at = torch.arange(p0 * page, p1 * page, device="cuda").view(-1, 1, page, 1)
            old = scales[pages]
            if pad[0] == 0:
                old[:] = 0
            else:
                old[1:] = 0
            top = (new.abs().amax((2, 3)).double() / 127).float()
            scale = torch.maximum(old, top)
            # next to a border between two codes a quotient of 32 bits may land on the wrong side
            wide = scale.double()[:, :, None, None]
            over = torch.where(wide > 0, wide, 1.0)
            was = codes[pages]
            moved = torch.where((at < first) & (wide > 0), torch.round(was.double() * old.double()[:, :, None, None] / over), was.double())
            fresh = torch.where(wide > 0, torch.round(new.double() / over), 0.0)
            codes[pages] = torch.where((at >= first) & (at < n), fresh, moved).clamp(-127, 127).to(torch.int8)
            scales[pages] = scale
    for out, codes, scales in zip(s["out"], (s["k"], s["v"]), (s["k_scale"], s["v_scale"])):
        for i, n in enumerate(s["host_lengths"]):
            b, e = s["back_starts"][i], s["back_starts"][i + 1]
            x = _plain_tokens(codes, scales, s["table"][i, (n - (e - b)) // page:-(-n // page)].long())[:, :e - b]
            out[b:e] = x.transpose(0, 1).reshape(e - b, heads * dim).to(out.dtype)
    return s["out"] + (s["k_scale"], s["v_scale"])


def _plain_verify(s):
    starts, tokens = s["starts"], s["tokens"].long()
    seqs = len(starts) - 1
    accepted, following = s["out"]
    place = torch.arange(seqs, device="cuda").repeat_interleave((s["offsets"][1:] - s["offsets"][:-1]).long(), output_size=starts[-1])
    mine = torch.arange(starts[-1], device="cuda")
    # whole probabilities of 32 bits: their products and sums need 64
    p = s["target"][mine + place, tokens].double()
    q = s["drafted"][mine, tokens].double() if s["drafted"] is not None else torch.ones_like(p)
    stands = s["accept"].double() * q < p
    for i in range(seqs):
        b, e = starts[i], starts[i + 1]
        n = torch.cumprod(stands[b:e].int(), 0).sum()
        row = s["target"][b + i:e + i + 1].index_select(0, n[None])[0].double()
        if e > b:
            at = torch.clamp(n, max=e - b - 1)
            less = torch.zeros_like(row)
            if s["drafted"] is not None:
                less = s["drafted"][b:e].index_select(0, at[None])[0].double()
            else:
                less[tokens[b + at]] = 1.0
            row = torch.where(n < e - b, torch.clamp(row - less, min=0.0), row)
        sums = torch.cumsum(row, 0)
        accepted[i] = n
        following[i] = (sums <= s["sample"][i].double() * sums[-1]).sum()
    return accepted, following


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _plain_attend, "append": _plain_append, "verify": _plain_verify}[state["case"]["kind"]](state)


def work(case):
    c = case
    if c["kind"] == "verify":
        n, cells = sum(_draft_counts(c)), c["seqs"] * c["vocab"]
        # of each sequence one row of the target's and one of the drafted probabilities, and single ones of the others
        return {"bytes": cells * BYTES[c["x"]] * (2 if c["drafted"] else 1) + 20 * n + 16 * c["seqs"], "flops": 3 * cells}
    new, lengths = _counts(c)
    heads, dim, page = c["kv_heads"], c["dim"], c["page"]
    token = 2 * heads * dim + 8 * heads / page                              # codes and scales of a cached token
    if c["kind"] == "append":
        back = sum(n - (n - m) // page * page for n, m in zip(lengths, new))
        rows = sum(new)
        # the new rows, their codes, what is read back, and what stood in pages that had been begun
        return {"bytes": rows * 2 * heads * dim * BYTES[c["x"]] + back * (token + 2 * heads * dim * BYTES[c["x"]]) + (back - rows) * token, "flops": 6 * rows * heads * dim}
    seen = touched = 0
    for n, m in zip(lengths, new):
        first = n - m
        if c["window"]:
            for p in range(first, n):
                low = max(0, p - c["window"] + 1)
                seen += p + 1 - low + min(c["sinks"], low)
            low = max(0, first - c["window"] + 1)
            touched += n - low + min(c["sinks"], low)
        else:
            seen += m * first + m * (m + 1) // 2
            touched += n
    return {"bytes": touched * token + 2 * sum(new) * c["heads"] * dim * BYTES[c["x"]], "flops": 4 * seen * c["heads"] * dim}


# --------------------------------------------------------------------------------------------- 64 bits
def _exact_attend(s):
    c = s["case"]
    if work(c)["flops"] > 2e13:
        return None
    kv_heads, dim, page = c["kv_heads"], c["dim"], c["page"]
    group = c["heads"] // kv_heads
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["host_lengths"]):
        b, e = s["starts"][i], s["starts"][i + 1]
        pages = s["table"][i, :-(-n // page)].long()
        j = torch.arange(n, device="cuda")
        where, slot = pages[j // page], j % page
        for h in range(kv_heads):
            k = s["k"][where, h, slot].to(torch.float64) * s["k_scale"][where, h].to(torch.float64).unsqueeze(1)
            v = s["v"][where, h, slot].to(torch.float64) * s["v_scale"][where, h].to(torch.float64).unsqueeze(1)
            for head in range(h * group, (h + 1) * group):
                for r in range(b, e, 2048):
                    t = min(e, r + 2048)
                    pos = torch.arange(n - e + r, n - e + t, device="cuda").unsqueeze(1)
                    hidden = j.unsqueeze(0) > pos
                    if c["window"]:
                        hidden |= (j.unsqueeze(0) <= pos - c["window"]) & (j.unsqueeze(0) >= c["sinks"])
                    x = torch.mm(s["q"][r:t, head * dim:(head + 1) * dim].to(torch.float64), k.t()).div_(math.sqrt(dim))
                    x[hidden] = -math.inf
                    out[r:t, head * dim:(head + 1) * dim] = torch.mm(torch.exp(x - torch.logsumexp(x, 1, keepdim=True)), v)
    return out


def _exact_append(s):
    c = s["case"]
    heads, dim, page = c["kv_heads"], c["dim"], c["page"]
    scales, outs = [], []
    for x, codes, scale in ((s["new_k"], s["k"], s["k_scale"].clone()), (s["new_v"], s["v"], s["v_scale"].clone())):
        out = torch.zeros(s["out"][0].shape, dtype=torch.float64, device="cuda")
        x = x.to(torch.float64).view(-1, heads, dim)
        for i, n in enumerate(s["host_lengths"]):
            b, at = s["starts"][i], s["back_starts"][i]
            m = s["starts"][i + 1] - b
            for start in range((n - m) // page * page, n, page):
                where = int(s["table"][i, start // page])
                lo, hi = max(start, n - m), min(start + page, n)
                mine = x[b + lo - (n - m):b + hi - (n - m)]
                before = scale[where].to(torch.float64) if lo > start else torch.zeros(heads, dtype=torch.float64, device="cuda")
                after = torch.maximum(before, (mine.abs().amax(dim=(0, 2)) / 127.0).to(torch.float32).to(torch.float64))      # a number of 32 bits
                safe = torch.where(after == 0, torch.ones_like(after), after).view(1, heads, 1)
                kept = codes[where, :, :lo - start].to(torch.float64).transpose(0, 1) * before.view(1, heads, 1)
                both = torch.cat([kept, mine]) / safe
                row = at + start - (n - m) // page * page
                out[row:row + hi - start] = (torch.round(both).clamp_(-127.0, 127.0) * after.view(1, heads, 1)).reshape(hi - start, heads * dim)
                scale[where] = after.to(torch.float32)
        outs.append(out)
        scales.append(scale.to(torch.float64))
    return tuple(outs) + tuple(scales)


def _exact_verify(s):
    count, last = [], []
    target, accept, sample = s["target"], s["accept"].tolist(), s["sample"].tolist()
    tokens = s["tokens"].tolist()
    for i in range(len(s["starts"]) - 1):
        b, e = s["starts"][i], s["starts"][i + 1]
        n = 0
        while b + n < e:
            p = float(target[b + i + n, tokens[b + n]])
            q = 1.0 if s["drafted"] is None else float(s["drafted"][b + n, tokens[b + n]])
            if not accept[b + n] * q < p:
                break
            n += 1
        mass = target[b + i + n].to(torch.float64)
        if b + n < e:
            if s["drafted"] is None:
                mass = mass.clone()
                mass[tokens[b + n]] = 0.0
            else:
                mass = torch.relu(mass - s["drafted"][b + n].to(torch.float64))
        upto = mass.cumsum(0)
        count.append(n)
        last.append(int(torch.searchsorted(upto, (upto[-1] * sample[i]).reshape(1), right=True)))
    return torch.tensor(count, dtype=torch.int32, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "verify": _exact_verify}[case["kind"]](s)
