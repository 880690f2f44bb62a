"""The operators of a decoder's step one after the other, with the int8 layers around them: a prompt, drafted tokens, tokens that were not taken back; streams, graphs and contexts."""
import numpy as np
import pytest

import decode_ops_reference as ref
import token_ops_reference as rows_ref

pytestmark = pytest.mark.gpu


class Decoder:
    """One layer: hidden states -> int8 projections -> cache -> attention -> logits -> probabilities -> which drafts stand."""

    def __init__(self, torch, zb, ctx, seqs, heads, kv_heads, dim, page, vocab, longest, seed, window=0, sinks=0):
        self.torch, self.ctx, self.window, self.sinks = torch, ctx, window, sinks
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.heads, self.kv_heads, self.dim, self.page, self.vocab, self.hidden = seqs, heads, kv_heads, dim, page, vocab, heads * dim
        wide = (heads + 2 * kv_heads) * dim
        self.w = {k: rng.integers(-127, 128, s, dtype=np.int8) for k, s in (("qkv", (wide, self.hidden)), ("head", (vocab, self.hidden)))}
        self.ws = {k: (rng.uniform(0.5, 1.5, len(v)) * 2.0 / (73 * np.sqrt(self.hidden))).astype(np.float32) for k, v in self.w.items()}
        self.dw, self.dws = ({k: torch.from_numpy(v).cuda() for k, v in d.items()} for d in (self.w, self.ws))
        width = -(-longest // page)
        pages = seqs * width + 2
        self.host = ref.Cache(pages, kv_heads, page, dim, rng)      # what pages held before
        self.cache = zb.KvCache(*[torch.from_numpy(x.copy()).cuda() for x in (self.host.codes[0], self.host.scales[0], self.host.codes[1], self.host.scales[1])])
        self.table = rng.permutation(pages)[:seqs * width].reshape(seqs, width).astype(np.int32)
        self.dtable = torch.from_numpy(self.table).cuda()

    def buffers(self, rows, drafts):
        t, d = self.torch, "cuda"
        wide = (self.heads + 2 * self.kv_heads) * self.dim
        return dict(x=t.zeros(rows, self.hidden, dtype=t.bfloat16, device=d), offsets=t.zeros(self.seqs + 1, dtype=t.int32, device=d), lengths=t.zeros(self.seqs, dtype=t.int32, device=d),
                    c=t.zeros(rows, self.hidden, dtype=t.int8, device=d), s=t.zeros(rows, device=d), qkv=t.zeros(rows, wide, dtype=t.bfloat16, device=d),
                    y=t.zeros(rows, self.hidden, dtype=t.bfloat16, device=d), c2=t.zeros(rows, self.hidden, dtype=t.int8, device=d), s2=t.zeros(rows, device=d),
                    logits=t.zeros(rows, self.vocab, device=d), p=t.zeros(rows, self.vocab, device=d), drafted=t.zeros(drafts, self.vocab, device=d),
                    tokens=t.zeros(drafts, dtype=t.int32, device=d), accept=t.zeros(drafts, device=d), sample=t.zeros(self.seqs, device=d),
                    accepted=t.zeros(self.seqs, dtype=t.int32, device=d), next=t.zeros(self.seqs, dtype=t.int32, device=d))

    def fill(self, b, new, lengths):
        """New inputs in place: hidden states, where they stand, random numbers, drafts."""
        rng, t = self.rng, self.torch
        put = lambda k, v: b[k].copy_(t.from_numpy(np.ascontiguousarray(v)))  # noqa: E731
        put("x", rng.standard_normal(tuple(b["x"].shape)).astype(np.float32))
        put("offsets", np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        put("lengths", np.asarray(lengths, np.int32))
        n = len(b["tokens"])
        p = rng.random((n, self.vocab)) ** 8
        put("drafted", (p / p.sum(1, keepdims=True)).astype(np.float32))
        put("tokens", rng.integers(0, self.vocab, n).astype(np.int32))
        put("accept", (rng.random(n) * 0.02).astype(np.float32))
        put("sample", rng.random(self.seqs).astype(np.float32))

    def run(self, b, verify=True):
        c, kv = self.ctx, self.heads * self.dim
        c.quantize_rows(b["x"], out=b["c"], out_scale=b["s"])
        c.qmatmul_scaled(b["c"], b["s"], self.dw["qkv"], self.dws["qkv"], out=b["qkv"])
        k, v = b["qkv"][:, kv:kv + self.kv_heads * self.dim], b["qkv"][:, kv + self.kv_heads * self.dim:]
        c.kv_cache_write(self.cache, k, v, self.dtable, b["lengths"], offsets=b["offsets"])
        c.kv_cache_attention(self.cache, b["qkv"][:, :kv], self.dtable, b["lengths"], offsets=b["offsets"], window=self.window, sinks=self.sinks, out=b["y"])
        c.quantize_rows(b["y"], out=b["c2"], out_scale=b["s2"])
        c.qmatmul_scaled(b["c2"], b["s2"], self.dw["head"], self.dws["head"], out=b["logits"])
        if verify:
            c.softmax(b["logits"], out=b["p"])
            c.verify_drafts(b["p"], b["drafted"], b["tokens"], b["accept"], b["sample"], out=(b["accepted"], b["next"]))

    def check(self, b, verify=True):
        """Every step against 64 bits of what the step before left."""
        g = {k: v.double().cpu().numpy() for k, v in b.items()}
        codes, scale = rows_ref.quantize_rows(g["x"])
        assert np.array_equal(g["c"], codes) and np.array_equal(g["s"].astype(np.float32), scale)
        want, off = rows_ref.scaled_product(codes, scale, self.w["qkv"], self.ws["qkv"], None, "bf16")
        assert (np.abs(g["qkv"] - want) <= off).all()
        rows, kv = len(g["x"]), self.heads * self.dim
        split = lambda x: x.reshape(rows, -1, self.dim)  # noqa: E731
        lengths, offsets = g["lengths"].astype(np.int64), g["offsets"].astype(np.int64)
        ref.write(self.host, [split(g["qkv"][:, kv:kv + self.kv_heads * self.dim]), split(g["qkv"][:, kv + self.kv_heads * self.dim:])], self.table, lengths, offsets)
        for have, codes, scales in ((self.cache.k, self.host.codes[0], None), (self.cache.v, self.host.codes[1], None), (self.cache.k_scale, None, self.host.scales[0]), (self.cache.v_scale, None, self.host.scales[1])):
            assert np.array_equal(have.cpu().numpy(), codes if scales is None else scales)
        want, off, _, _, there = ref.attention(self.host, split(g["qkv"][:, :kv]), self.table, lengths, offsets, "bf16", None, self.window, self.sinks)
        assert there.all() and (np.abs(split(g["y"]) - want) <= off).all()
        codes, scale = rows_ref.quantize_rows(g["y"])
        assert np.array_equal(g["c2"], codes)
        want, off = rows_ref.scaled_product(codes, scale, self.w["head"], self.ws["head"], None, "f32")
        assert (np.abs(g["logits"] - want) <= off).all()
        if verify:
            n, following = ref.verify(g["p"], g["drafted"], b["tokens"].cpu().numpy(), b["accept"].cpu().numpy(), b["sample"].cpu().numpy(), None)
            assert np.array_equal(g["accepted"], n) and np.array_equal(g["next"], following)
            return n


@pytest.mark.parametrize("heads,kv_heads,dim,page,window,sinks", [(8, 2, 64, 16, 0, 0), (6, 3, 128, 32, 40, 4), (4, 4, 80, 64, 0, 0), (2, 1, 256, 16, 100, 0)])
def test_a_prompt_and_drafts(ctx, zb, heads, kv_heads, dim, page, window, sinks):
    """Three sequences: prompts of different lengths, then drafted tokens; those that do not stand are written over by the next step's."""
    import torch
    d = Decoder(torch, zb, ctx, 3, heads, kv_heads, dim, page, 700, 400, dim + page, window, sinks)
    new = [90, 1, 200]
    b = d.buffers(sum(new), 0)
    d.fill(b, new, new)
    torch.cuda.synchronize()
    d.run(b, verify=False)
    ctx.synchronize()
    d.check(b, verify=False)
    lengths, drafts = np.array(new), 3
    b = d.buffers(3 * (drafts + 1), 3 * drafts)
    for _ in range(6):
        d.fill(b, [drafts + 1] * 3, lengths + drafts + 1)
        torch.cuda.synchronize()
        d.run(b)
        ctx.synchronize()
        lengths = lengths + d.check(b) + 1


def test_captured_and_replayed(zb):
    """Two decoders on one context, their steps captured and replayed in turn on other tokens, lengths and random numbers, beside eager calls."""
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    sets = []
    for i, (heads, kv_heads, dim, page, rows) in enumerate(((8, 2, 128, 32, 2), (4, 1, 64, 16, 70))):
        d = Decoder(torch, zb, c, 2, heads, kv_heads, dim, page, 300, 600, i)
        sets.append((d, d.buffers(2 * rows, 2 * (rows - 1)), rows))
    eager = Decoder(torch, zb, c, 2, 4, 4, 96, 64, 200, 300, 7)
    eb = eager.buffers(2 * 3, 2 * 2)
    torch.cuda.synchronize()
    graphs = []
    for d, b, rows in sets:
        d.fill(b, [rows] * 2, [rows + 5, rows + 9])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream, capture_error_mode="thread_local"):
            d.run(b)
    for turn in range(3):
        for d, b, rows in sets:
            d.fill(b, [rows] * 2, [rows + 7 + 100 * turn, rows + 3 * turn])
        eager.fill(eb, [3, 3], [20 + turn, 3])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay()
            eager.run(eb)
            graphs[1].replay()
        torch.cuda.synchronize()
        for d, b in [s[:2] for s in sets] + [(eager, eb)]:
            d.check(b)
    stream.synchronize()
    del graphs
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_captured_long_context_needs_no_workspace(zb):
    """Few tiles of a long context: the workspace that an eager call takes is no part of a graph."""
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(1)
    cache = ref.Cache(20000 // 64 + 2, 1, 64, 64, rng)
    held = zb.KvCache(*[torch.from_numpy(x).cuda() for x in (cache.codes[0], cache.scales[0], cache.codes[1], cache.scales[1])])
    table = rng.permutation(20000 // 64 + 2)[None, :313].astype(np.int32)
    q = torch.randn(1, 4 * 64, device="cuda")
    t, n, y = torch.from_numpy(table).cuda(), torch.tensor([20000], dtype=torch.int32, device="cuda"), [torch.zeros(1, 4 * 64, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        c.kv_cache_attention(held, q, t, n, out=y[0])
        assert c.last_kernel() == "kv_attention_kernel"
    c.kv_cache_attention(held, q, t, n, out=y[1])
    assert c.last_kernel() == "kv_attention_join_kernel"
    for length in (20000, 700, 0, 13000):
        n.fill_(length)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        c.kv_cache_attention(held, q, t, n, out=y[1])
        torch.cuda.synchronize()
        want, off, _, _, _ = ref.attention(cache, q.double().cpu().numpy().reshape(1, 4, 64), table, [length], None, "f32")
        for got in y:
            assert (np.abs(got.double().cpu().numpy().reshape(1, 4, 64) - want) <= off).all()
    del graph
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_each_call_with_host_operands_is_refused_in_a_capture(zb):
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    arrays = [np.zeros((2, 1, 16, 32), np.int8), np.ones((2, 1), np.float32), np.zeros((2, 1, 16, 32), np.int8), np.ones((2, 1), np.float32)]
    host, dev = zb.KvCache(*arrays), zb.KvCache(*[torch.from_numpy(a).cuda() for a in arrays])
    x, y, table, lengths = torch.ones(1, 32, device="cuda"), torch.zeros(1, 32, device="cuda"), i(1)[None], i(5)
    p, n, f = torch.full((2, 8), 0.125, device="cuda"), i(0), i(0)
    hx, ht, hn, u = np.ones((1, 32), np.float32), np.ones((1, 1), np.int32), np.array([5], np.int32), torch.full((1,), 0.5, device="cuda")
    refused = [lambda: c.kv_cache_write(host, x, x, table, lengths), lambda: c.kv_cache_write(dev, hx, x, table, lengths), lambda: c.kv_cache_write(dev, x, x, ht, lengths),
               lambda: c.kv_cache_write(dev, x, x, table, hn), lambda: c.kv_cache_write(dev, x, x, table, lengths, offsets=[0, 1]), lambda: c.kv_cache_read(host, table, lengths, out=(y, None)),
               lambda: c.kv_cache_read(dev, table, lengths, out=(None, hx)), lambda: c.kv_cache_attention(host, x, table, lengths, out=y), lambda: c.kv_cache_attention(dev, hx, table, lengths, out=y),
               lambda: c.kv_cache_attention(dev, x, table, hn, out=y), lambda: c.kv_cache_attention(dev, x, table, lengths, out=y, lse=np.zeros((1, 1), np.float32)),
               lambda: c.verify_drafts(p, None, [3], u, u, out=(n, f)), lambda: c.verify_drafts(p, None, drafts, np.ones(1, np.float32), u, out=(n, f)),
               lambda: c.verify_drafts(p, np.ones((1, 8), np.float32), drafts, u, u, out=(n, f)), lambda: c.verify_drafts(p, None, drafts, u, u, out=(np.zeros(1, np.int32), f))]
    drafts = i(3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        c.kv_cache_write(dev, x, x, table, lengths)
        for call in refused:
            with pytest.raises(zb.ZantError) as e:
                call()
            assert "cannot be captured" in str(e.value)
        c.kv_cache_attention(dev, x, table, lengths, out=y, sinks=0, window=1)
        c.verify_drafts(p, None, drafts, u, u, out=(n, f))
    torch.cuda.synchronize()
    assert (y == 0).all() and int(dev.k.abs().sum()) == 0
    graph.replay()
    torch.cuda.synchronize()
    # the window holds the token itself: its values, 127 times a scale of 1 / 127 that was rounded once
    assert ((y.double() - 1).abs() <= 4 * ref.U).all() and int(n[0]) == 0 and int(f[0]) == 4
    del graph
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_two_contexts_on_streams_of_their_own(zb):
    import torch
    parts = []
    for i in range(2):
        c, stream = zb.Context(0), torch.cuda.Stream()
        c.set_stream(stream.cuda_stream)
        d = Decoder(torch, zb, c, 2, 8, 2, 128, 32, 500, 500, 30 + i)
        rows = (4, 90)[i]
        b = d.buffers(2 * rows, 2 * (rows - 1))
        d.fill(b, [rows] * 2, [rows + 11, rows + 300])
        parts.append((c, d, b))
    torch.cuda.synchronize()
    for _ in range(10):                               # (a step again on the same tokens leaves what it left)
        for c, d, b in parts:
            d.run(b)
    for c, d, b in parts:
        c.synchronize()
        d.check(b)
        c.set_stream(torch.cuda.default_stream().cuda_stream)
        c.close()


def test_launches_are_counted(ctx, zb):
    import torch
    d = Decoder(torch, zb, ctx, 2, 4, 2, 64, 16, 100, 100, 3)
    b = d.buffers(4, 2)
    d.fill(b, [2, 2], [9, 30])
    torch.cuda.synchronize()
    before = ctx.launch_count()
    d.run(b)
    ctx.synchronize()
    assert ctx.launch_count() - before == 8
