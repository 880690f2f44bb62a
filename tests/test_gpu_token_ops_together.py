"""The language-model operators one after the other, as a decoder would call them, and how they share streams and graphs."""
import numpy as np
import pytest

import token_ops_reference as ref

pytestmark = pytest.mark.gpu


class Block:
    """Hidden states -> experts with a gated activation -> logits -> log probabilities, on int8 weights."""

    def __init__(self, torch, ctx, tokens, hidden, inner, experts, top, vocab, seed):
        self.torch, self.ctx, self.top = torch, ctx, top
        rng = np.random.default_rng(seed)
        self.shape = (tokens, hidden, inner, experts, vocab)
        host = dict(up=rng.integers(-127, 128, (experts, inner, hidden), dtype=np.int8), gate=rng.integers(-127, 128, (experts, inner, hidden), dtype=np.int8),
                    down=rng.integers(-127, 128, (experts, hidden, inner), dtype=np.int8), head=rng.integers(-127, 128, (vocab, hidden), dtype=np.int8))
        host |= {k + "_s": (rng.uniform(0.5, 1.5, v.shape[:-1]) / (73 * np.sqrt(v.shape[-1]))).astype(np.float32) for k, v in list(host.items())}
        chosen = np.stack([rng.permutation(experts)[:top] for _ in range(tokens)]).reshape(-1)
        order = np.argsort(chosen, kind="stable")
        host["index"] = (order // top).astype(np.int32)
        host["offsets"] = np.concatenate([[0], np.cumsum(np.bincount(chosen, minlength=experts))]).astype(np.int32)
        host["x"] = rng.standard_normal((tokens, hidden)).astype(np.float32)
        host["given"] = rng.integers(0, vocab, tokens * top).astype(np.int32)
        self.host = host
        self.dev = {k: torch.from_numpy(v).cuda() for k, v in host.items()}
        rows = tokens * top
        f = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        i = lambda *s: torch.empty(*s, dtype=torch.int8, device="cuda")  # noqa: E731
        self.buf = dict(q=i(rows, hidden), s=f(rows), up=f(rows, inner), gate=f(rows, inner), sig=f(rows, inner), q2=i(rows, inner), s2=f(rows), out=f(rows, hidden),
                        q3=i(rows, hidden), s3=f(rows), logits=torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda"),
                        lp=f(rows), h=f(rows), ids=torch.empty(rows, 5, dtype=torch.int32, device="cuda"), tlp=f(rows, 5))

    def run(self):
        c, d, b = self.ctx, self.dev, self.buf
        c.quantize_rows(d["x"], index=d["index"], out=b["q"], out_scale=b["s"])
        c.qmatmul_grouped(b["q"], b["s"], d["up"], d["up_s"], d["offsets"], out=b["up"])
        c.qmatmul_grouped(b["q"], b["s"], d["gate"], d["gate_s"], d["offsets"], out=b["gate"])
        c.sigmoid(b["gate"], out=b["sig"])
        c.mul(b["gate"], b["sig"], out=b["sig"])
        c.mul(b["sig"], b["up"], out=b["up"])
        c.quantize_rows(b["up"], out=b["q2"], out_scale=b["s2"])
        c.qmatmul_grouped(b["q2"], b["s2"], d["down"], d["down_s"], d["offsets"], out=b["out"])
        c.quantize_rows(b["out"], out=b["q3"], out_scale=b["s3"])
        c.qmatmul_scaled(b["q3"], b["s3"], d["head"], d["head_s"], out=b["logits"])
        c.token_logprobs(b["logits"], d["given"], top=5, out=(b["lp"], b["h"], b["ids"], b["tlp"]))

    def check(self):
        """Every step against 64 bits of what the step before left (the errors of one step do not blur the next)."""
        h, g = self.host, {k: v.double().cpu().numpy() for k, v in self.buf.items()}
        x = self.dev["x"].double().cpu().numpy()

        def same_codes(q, s, x, index=None):
            wq, ws = ref.quantize_rows(x, index)
            assert np.array_equal(g[q], wq) and np.array_equal(g[s].astype(np.float32), ws)

        def product(y, q, s, name, t):
            for e in range(self.shape[3]) if h[name].ndim == 3 else [None]:
                r = slice(None) if e is None else slice(h["offsets"][e], h["offsets"][e + 1])
                w, ws = (h[name], h[name + "_s"]) if e is None else (h[name][e], h[name + "_s"][e])
                want, off = ref.scaled_product(g[q][r].astype(np.int8), g[s][r].astype(np.float32), w, ws, None, t)
                assert (np.abs(g[y][r] - want) <= off).all()
        same_codes("q", "s", x, h["index"])
        product("gate", "q", "s", "gate", "f32")
        same_codes("q2", "s2", g["up"])
        product("out", "q2", "s2", "down", "f32")
        same_codes("q3", "s3", g["out"])
        product("logits", "q3", "s3", "head", "bf16")
        given, entropy, ids, likely = ref.token_logprobs(g["logits"], h["given"], 5)
        log_s, off = ref.logprob_bound(g["logits"])
        assert (np.abs(g["lp"] - given) <= log_s + 4 * ref.U * (1 + np.abs(given))).all()
        assert (np.abs(g["h"] - entropy) <= off).all()
        assert np.array_equal(g["ids"], ids) and (np.abs(g["tlp"] - likely) <= log_s[:, None] + 4 * ref.U * (1 + np.abs(likely))).all()


@pytest.mark.parametrize("tokens,hidden,inner,experts,top,vocab", [(1, 256, 128, 8, 2, 1000), (37, 320, 208, 5, 3, 4001), (300, 512, 256, 16, 4, 9000)])
def test_block(ctx, tokens, hidden, inner, experts, top, vocab):
    import torch
    b = Block(torch, ctx, tokens, hidden, inner, experts, top, vocab, tokens)
    torch.cuda.synchronize()
    b.run()
    ctx.synchronize()
    b.check()


def test_captured_and_replayed(zb):
    """Two graphs of different sizes on one context, replayed in turn on new inputs, beside eager calls of the same operators."""
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    blocks = [Block(torch, c, 3, 256, 144, 6, 2, 1500, 1), Block(torch, c, 70, 512, 256, 4, 2, 3000, 2)]
    torch.cuda.synchronize()
    graphs = []
    for b in blocks:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream, capture_error_mode="thread_local"):
            b.run()
    eager = Block(torch, c, 20, 256, 128, 4, 2, 800, 3)
    for turn in range(3):
        for b in blocks:
            b.dev["x"].mul_(1.0 + turn).add_(0.01)
            for v in b.buf.values():
                v.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay()
            graphs[1].replay()
            eager.run()
        torch.cuda.synchronize()
        for b in blocks + [eager]:
            b.check()
    stream.synchronize()
    del graphs
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_host_arrays_are_refused_in_a_capture(zb):
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    x = torch.ones(4, 64, device="cuda")
    q, s = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        c.quantize_rows(x, out=q, out_scale=s)
        for call in (lambda: c.quantize_rows(np.ones((4, 64), np.float32), out=q, out_scale=s), lambda: c.qmatmul_scaled(q, s, np.ones((5, 64), np.int8), np.ones(5, np.float32), out=torch.zeros(0)[:0].view(0, 0)),
                     lambda: c.token_logprobs(x, [1, 2, 3, 4])):
            with pytest.raises(zb.ZantError):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert (q == 127).all()
    del graph
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_two_contexts_on_streams_of_their_own(zb):
    """Two programs at once: contexts share nothing."""
    import torch
    parts = []
    for i in range(2):
        c, stream = zb.Context(0), torch.cuda.Stream()
        c.set_stream(stream.cuda_stream)
        parts.append((c, stream, Block(torch, c, 40 + 90 * i, 512, 256, 8, 2, 2500, 20 + i)))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, stream, b in parts:
            b.run()
    for c, stream, b in parts:
        c.synchronize()
        b.check()
        c.set_stream(torch.cuda.default_stream().cuda_stream)
        c.close()


def test_launches_are_counted(ctx):
    import torch
    b = Block(torch, ctx, 5, 128, 64, 4, 2, 500, 9)
    torch.cuda.synchronize()
    before = ctx.launch_count()
    b.run()
    ctx.synchronize()
    assert ctx.launch_count() - before == 11


def test_each_call_with_host_operands_is_refused_in_a_capture(zb):
    """With results of the right size on the device, so that nothing but the host operand is refused, by the library and with its reason."""
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    x = torch.ones(4, 64, device="cuda")
    q, s = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    w, ws, off = torch.ones(5, 64, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    y, lp, h, none = torch.full((4, 5), 7.0, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), (torch.zeros(4, 0, dtype=torch.int32, device="cuda"), torch.zeros(4, 0, device="cuda"))
    ones = np.ones
    refused = [lambda: c.quantize_rows(ones((4, 64), np.float32), out=q, out_scale=s), lambda: c.quantize_rows(x, index=[0, 1, 2, 3], out=q, out_scale=s),
               lambda: c.qmatmul_scaled(q, s, ones((5, 64), np.int8), ws, out=y), lambda: c.qmatmul_scaled(ones((4, 64), np.int8), s, w, ws, out=y),
               lambda: c.qmatmul_scaled(q, s, w, ones(5, np.float32), out=y), lambda: c.qmatmul_scaled(q, s, w, ws, out=torch.zeros(4, 5)),
               lambda: c.qmatmul_grouped(q, s, w[None], ws[None], [0, 4], out=y), lambda: c.token_logprobs(x, [1, 2, 3, 4], out=(lp, h) + none)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        c.quantize_rows(x, out=q, out_scale=s)
        for call in refused:
            with pytest.raises(zb.ZantError) as e:
                call()
            assert "cannot be captured" in str(e.value)
        c.qmatmul_grouped(q, s, w[None], ws[None], off, out=y)
    torch.cuda.synchronize()
    assert (y == 7).all()
    graph.replay()
    torch.cuda.synchronize()
    # sums of 64 * 127, times a scale of 1 / 127 that was rounded once, and two products that round once each
    assert ((y.double() - 64.0).abs() <= 64 * 3.1 * ref.U).all()
    del graph
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()
