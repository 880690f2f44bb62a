"""The kernels behind qmatmul_scaled and qmatmul_grouped that sizes and addresses choose between, each at sizes where its tiles end inside."""
import numpy as np
import pytest

import token_ops_reference as ref
from test_gpu_scaled_products import check, check_groups, grouped, operands, place, product, torch_type

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tight(zb):
    """A context whose arena has no room to lay operands out: rows at odd addresses are read where they are."""
    c = zb.Context(0, arena_bytes=4096)
    yield c
    c.close()


def sampled(torch, y, ops, t, count=60):
    """Rows and columns of every part of a large product, against 64 bits."""
    rng = np.random.default_rng(1)
    rows, n = y.shape
    r = np.unique(np.concatenate([np.arange(min(rows, 4)), rng.integers(0, rows, count), np.arange(max(0, rows - 4), rows)]))
    c = np.unique(np.concatenate([np.arange(min(n, 4)), rng.integers(0, n, 3 * count), np.arange(max(0, n - 4), n)]))
    check(y[torch.from_numpy(r).cuda()][:, torch.from_numpy(c).cuda()], ops[0][r], ops[1][r], ops[2][c], ops[3][c], None if ops[4] is None else ops[4][c], t)


@pytest.mark.parametrize("rows,k,n,t", [
    (8, 4096, 4100, "bf16"), (16, 1000, 2049, "f16"),                       # few tokens
    (16, 512, 19000, "f32"), (64, 2048, 1030, "bf16"),                      # 64 columns
    (257, 640, 5008, "f16"), (130, 320, 9001, "f32"),                       # 128
    (38000, 64, 128, "bf16"), (37900, 160, 100, "f16"),                     # 256, one tile of channels
    (1000, 512, 4096, "bf16"), (2050, 272, 4000, "f32"), (4099, 144, 3333, "f16"), (777, 1040, 8191, "bf16")])        # pairs of CTAs
def test_sizes_of_each_kernel(ctx, rows, k, n, t):
    import torch
    ops = operands(np.random.default_rng(rows), rows, k, n, bias=rows % 2 == 0)
    pad = -k % 16
    sampled(torch, product(ctx, torch, *ops, t, (0, pad), (0, pad)), ops, t)


@pytest.mark.parametrize("rows,k,n,t", [
    (40, 9033, 1856, "bf16"), (113, 9792, 1472, "f16"), (17, 4000, 129, "f32"), (128, 5000, 33, "bf16"),                  # few tiles with a long k
    (777, 1040, 8191, "f16"), (420, 144, 6200, "f32"), (449, 160, 6300, "bf16"), (1116, 272, 11328, "bf16"), (300, 80, 6331, "f16"), (385, 144, 8000, "f32")])  # pairs whose last tiles are short
def test_long_rows_and_last_pairs(ctx, rows, k, n, t):
    import torch
    ops = operands(np.random.default_rng(rows), rows, k, n, bias=rows % 2 == 0)
    pad = -k % 16
    sampled(torch, product(ctx, torch, *ops, t, (0, pad), (0, pad)), ops, t)


@pytest.mark.parametrize("counts", [[340, 300], [0, 900, 131, 65], [257, 5, 640]])
@pytest.mark.parametrize("k,n,a_at,w_at", [(77, 200, (0, 0), (0, 0)), (513, 129, (0, 15), (0, 0)), (400, 300, (1, 0), (0, 0)), (400, 2900, (0, 0), (0, 0))])
def test_longer_groups(ctx, tight, counts, k, n, a_at, w_at):
    import torch
    offsets = np.concatenate([[1], 1 + np.cumsum(counts)])
    ops = operands(np.random.default_rng(k + n), int(offsets[-1]) + 3, k, n, len(counts), bias=True)
    for c in (ctx, tight):
        check_groups(grouped(c, torch, ops, offsets, "bf16", 2, a_at, w_at), ops, offsets, "bf16")


@pytest.mark.parametrize("a_at,w_at", [((0, 0), (1, 0)), ((7, 0), (0, 0)), ((3, 1), (5, 2)), ((1, 4), (2, 6))])
@pytest.mark.parametrize("rows,k,n", [(3, 700, 130), (30, 333, 257), (33, 129, 128), (129, 1001, 300), (260, 64, 129), (70, 4111, 131)])
def test_rows_read_where_they_are(tight, rows, k, n, a_at, w_at):
    import torch
    ops = operands(np.random.default_rng(rows + k), rows, k, n, bias=True)
    for t in ("f32", "bf16"):
        check(product(tight, torch, *ops, t, a_at, w_at), *ops, t)


@pytest.mark.parametrize("counts", [[40, 0, 129, 1, 260], [200, 33], [128] * 5])
@pytest.mark.parametrize("k,n,a_at,w_at", [(77, 200, (0, 0), (0, 0)), (513, 129, (0, 15), (0, 0)), (400, 300, (1, 0), (0, 0))])
def test_groups_read_where_they_are(tight, counts, k, n, a_at, w_at):
    import torch
    offsets = np.concatenate([[3], 3 + np.cumsum(counts)])
    ops = operands(np.random.default_rng(k), int(offsets[-1]) + 2, k, n, len(counts), bias=True)
    check_groups(grouped(tight, torch, ops, offsets, "f16", 1, a_at, w_at), ops, offsets, "f16")


def test_laid_out_and_read_in_place_agree(ctx, tight):
    import torch
    ops = operands(np.random.default_rng(5), 150, 1999, 401, bias=True)
    y = [product(c, torch, *ops, "f32", a_at, w_at) for c in (ctx, tight) for a_at, w_at in (((0, 0), (0, 0)), ((1, 0), (0, 3)), ((0, 1), (0, 1)))]
    assert all(torch.equal(y[0], v) for v in y[1:])


def test_calls_in_a_row_share_the_arena(ctx):
    """Operands laid out for one product are not overwritten by the next call's before it has read them."""
    import torch
    rng = np.random.default_rng(6)
    work = []
    for i in range(12):
        ops = operands(rng, 300 + 7 * i, 1001 + 2 * i, 600 + i)
        dev = [place(torch, ops[0], i % 3), torch.from_numpy(ops[1]).cuda(), place(torch, ops[2], i % 2), torch.from_numpy(ops[3]).cuda()]
        work.append((ops, dev, torch.empty(ops[0].shape[0], ops[2].shape[0], device="cuda")))
    torch.cuda.synchronize()
    for _ops, dev, y in work:
        ctx.qmatmul_scaled(*dev, out=y)
    ctx.synchronize()
    for ops, _dev, y in work:
        sampled(torch, y, ops, "f32", 20)


def test_each_kernel_in_a_graph(zb):
    """Captured: few tokens, tiles of 64, pairs of CTAs, rows at odd addresses (which are read where they are then), replayed on new values."""
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(7)
    work = []
    for rows, k, n, off in ((4, 512, 300, 0), (60, 512, 3000, 0), (1100, 256, 4096, 0), (200, 511, 700, 1), (5, 333, 100, 3), (140, 640, 513, 7)):
        ops = operands(rng, rows, k, n)
        dev = [place(torch, ops[0], off), torch.from_numpy(ops[1]).cuda(), place(torch, ops[2], off), torch.from_numpy(ops[3]).cuda()]
        work.append([ops, dev, torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        for _ops, dev, y in work:
            c.qmatmul_scaled(*dev, out=y)
    for turn in range(2):
        for w in work:
            a = rng.integers(-127, 128, w[0][0].shape, dtype=np.int8)
            w[0] = (a,) + w[0][1:]
            w[1][0].copy_(torch.from_numpy(a))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for ops, _dev, y in work:
            sampled(torch, y, ops, "bf16", 30)
    del graph
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_streams_in_turn(zb):
    """One context moved from stream to stream: each call's results are right, also those that use the arena."""
    import torch
    c = zb.Context(0)
    streams = [torch.cuda.Stream() for _ in range(3)]
    ops = operands(np.random.default_rng(8), 170, 1003, 333)
    dev = [torch.from_numpy(v).cuda() for v in ops[:4]]
    ys = [torch.empty(170, 333, device="cuda") for _ in range(9)]
    torch.cuda.synchronize()
    for i, y in enumerate(ys):
        c.set_stream(streams[i % 3].cuda_stream)
        c.qmatmul_scaled(*dev, out=y)
    c.synchronize()
    torch.cuda.synchronize()
    for y in ys:
        check(y, *ops[:4], None, "f32")
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_arena_limit_and_host_operands(zb):
    """Host operands beyond the arena's limit are refused, and the context works on; with room they give the same bits as device operands."""
    import torch
    rng = np.random.default_rng(9)
    ops = operands(rng, 90, 777, 300)
    want, off = ref.scaled_product(*ops, "f32")
    with zb.Context(0, arena_bytes=1 << 16) as c:
        c.set_arena_limit(1 << 17)
        with pytest.raises(zb.ZantError) as e:
            c.qmatmul_scaled(*ops[:4])
        assert e.value.name == "ArenaExhausted"
        c.set_arena_limit(0)
        host = c.qmatmul_scaled(*ops[:4])
        assert (np.abs(host - want) <= off).all()
        y = torch.empty(90, 300, device="cuda")
        c.qmatmul_scaled(*[torch.from_numpy(v).cuda() for v in ops[:4]], out=y)
        c.synchronize()
        assert np.array_equal(y.cpu().numpy(), host)
        # host results in rows further apart than they are long: what lies between stays
        room = torch.full((90, 320), 5.0)
        c.qmatmul_scaled(*ops[:4], out=room[:, :300])
        assert (room[:, 300:] == 5).all() and np.array_equal(room[:, :300].numpy(), host)
