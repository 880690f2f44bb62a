"""Which kernel sizes and addresses choose behind qmatmul_scaled and qmatmul_grouped: each is run, by name, dense and grouped, and in a captured graph."""
import numpy as np
import pytest

from test_gpu_scaled_kernels import sampled
from test_gpu_scaled_products import check_groups, grouped, operands, place, product

pytestmark = pytest.mark.gpu
FEW, ANY, PAIR = "scaled_few_kernel", "scaled_any_kernel", "scaled_pair_kernel"
GEMM = {nt: f"scaled_gemm_kernel<{nt}>" for nt in (64, 128, 256)}


@pytest.fixture(scope="module")
def tight(zb):
    """A context whose arena has no room to lay operands out: rows at odd addresses are read where they are."""
    c = zb.Context(0, arena_bytes=4096)
    yield c
    c.close()


@pytest.mark.parametrize("rows,k,n,t,kernel", [
    (8, 4096, 4100, "bf16", FEW), (64, 2048, 1030, "f16", FEW), (113, 1040, 900, "f32", FEW),
    (16, 512, 19000, "f32", GEMM[64]), (113, 9792, 1472, "f16", GEMM[64]), (60, 144, 3001, "bf16", GEMM[64]),
    (257, 640, 5008, "f16", GEMM[128]), (38000, 64, 128, "bf16", GEMM[128]), (1100, 256, 4096, "f32", GEMM[128]),
    (700, 144, 6200, "bf16", GEMM[256]), (20000, 64, 128, "f16", GEMM[256]), (700, 1040, 6200, "f32", GEMM[256]), (19100, 528, 97, "f32", GEMM[256]),
    (753, 1040, 6111, "f32", PAIR), (1000, 512, 4096, "bf16", PAIR), (2050, 272, 4000, "f32", PAIR), (777, 1040, 8191, "f16", PAIR)])
def test_dense(ctx, rows, k, n, t, kernel):
    import torch
    ops = operands(np.random.default_rng(rows), rows, k, n, bias=rows % 2 == 0)
    pad = -k % 16
    y = product(ctx, torch, *ops, t, (0, pad), (0, pad))
    assert ctx.last_kernel() == kernel
    sampled(torch, y, ops, t)


@pytest.mark.parametrize("rows,k,n,groups,kernel", [
    (20, 1040, 320, 4, FEW), (470, 320, 2000, 5, GEMM[64]), (6000, 128, 256, 16, GEMM[128]), (5691, 144, 541, 20, GEMM[256]), (1300, 144, 2500, 4, PAIR)])
@pytest.mark.parametrize("skewed", [False, True])
def test_grouped(ctx, rows, k, n, groups, kernel, skewed):
    """Groups of about the same size, and nearly all rows in one of them."""
    import torch
    rng = np.random.default_rng(rows + skewed)
    inner = np.sort(rng.integers(2, 12 if skewed else rows - 3, groups - 1))
    offsets = np.concatenate([[1], inner, [rows - 2]])
    ops = operands(rng, rows, k, n, groups, bias=skewed)
    y = grouped(ctx, torch, ops, offsets, "f32")
    assert ctx.last_kernel() == kernel
    check_groups(y, ops, offsets, "f32")


@pytest.mark.parametrize("rows,k,n,off,kernel", [(30, 333, 257, 1, FEW), (128, 1001, 300, 3, FEW), (129, 1001, 300, 3, ANY), (140, 640, 513, 7, ANY), (300, 999, 1030, 1, ANY)])
def test_rows_read_where_they_are(tight, rows, k, n, off, kernel):
    import torch
    ops = operands(np.random.default_rng(rows), rows, k, n)
    for a_at, w_at in (((off, 0), (off, 0)), ((off, 0), (0, -k % 16)), ((0, -k % 16), (off, 0))):
        y = product(tight, torch, *ops, "f16", a_at, w_at)
        assert tight.last_kernel() == kernel
        sampled(torch, y, ops, "f16")


@pytest.mark.parametrize("groups,rows,n", [(16, 528, 256), (30, 990, 128)])
def test_groups_at_odd_addresses_are_laid_out(ctx, tight, groups, rows, n):
    """Groups of 33 rows: few tiles if they lay side by side, too many for the few-token kernel as groups.  Where the arena has room they are laid out."""
    import torch
    k = 1001
    offsets = np.arange(groups + 1) * 33
    ops = operands(np.random.default_rng(rows), rows, k, n, groups)
    y = grouped(ctx, torch, ops, offsets, "f32")
    assert ctx.last_kernel() in GEMM.values()
    check_groups(y, ops, offsets, "f32")
    there = grouped(tight, torch, ops, offsets, "f32")
    assert tight.last_kernel() == ANY and torch.equal(y, there)


def test_in_a_graph(zb):
    """Each kernel captured, pairs of CTAs among them, and replayed on new values."""
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(7)
    work = []
    for rows, k, n, off, kernel in ((4, 512, 300, 0, FEW), (60, 512, 3000, 0, GEMM[64]), (1100, 256, 4096, 0, GEMM[128]), (1000, 512, 4096, 0, PAIR), (700, 144, 6200, 0, GEMM[256]),
                                    (2050, 272, 4000, 0, PAIR), (200, 511, 700, 1, ANY), (5, 333, 100, 3, FEW)):
        ops = operands(rng, rows, k, n)
        dev = [place(torch, ops[0], off), torch.from_numpy(ops[1]).cuda(), place(torch, ops[2], off), torch.from_numpy(ops[3]).cuda()]
        work.append([ops, dev, torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda"), kernel])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        for _ops, dev, y, kernel in work:
            c.qmatmul_scaled(*dev, out=y)
            assert c.last_kernel() == kernel
    for turn in range(3):
        for w in work:
            a = rng.integers(-127, 128, w[0][0].shape, dtype=np.int8)
            w[0] = (a,) + w[0][1:]
            w[1][0].copy_(torch.from_numpy(a))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for ops, _dev, y, _kernel in work:
            sampled(torch, y, ops, "bf16", 30)
    c.synchronize()
    del graph
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()


def test_name_before_the_first_launch(zb):
    with zb.Context(0) as c:
        assert c.last_kernel() == ""


def test_a_host_result_beside_rows_to_lay_out(zb):
    """An arena that holds the host result but not the operands as well: they are read where they are, and a limit on the arena refuses nothing."""
    import torch
    rows, k, n = 200, 999, 300
    ops = operands(np.random.default_rng(21), rows, k, n)
    dev = [torch.from_numpy(v).cuda() for v in ops[:4]]
    torch.cuda.synchronize()
    laid_out = (rows + n) * 1008 + 512
    size = max(laid_out, rows * n * 4 + 256) + 4096        # either has room, both have not
    with zb.Context(0, arena_bytes=size) as c:
        c.set_arena_limit(size)
        y = torch.zeros(rows, n, device="cuda")
        torch.cuda.synchronize()
        c.qmatmul_scaled(*dev, out=y)
        assert c.last_kernel() in GEMM.values()
        c.synchronize()
        host = c.qmatmul_scaled(*dev)
        assert c.last_kernel() == ANY and np.array_equal(host, y.cpu().numpy())
        sampled(torch, y, ops, "f32")
