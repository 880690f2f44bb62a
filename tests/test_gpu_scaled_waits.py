"""Waits of the tcgen05 kernels behind qmatmul_scaled and qmatmul_grouped that run out: a CTA gives up on the healthy GPU, every warp of it (and the other CTA
of its pair) comes to the kernel's end, the call reports the time-out, and the products behind it are right."""
import numpy as np
import pytest

from test_gpu_scaled_kernels import sampled
from test_gpu_scaled_products import check_groups, grouped, operands, product

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tight(zb):
    """A context whose arena has no room to lay operands out: rows at odd addresses are read where they are."""
    c = zb.Context(0, arena_bytes=4096)
    yield c
    c.close()


def timed_out(zb, call):
    with pytest.raises(zb.ZantError) as e:
        call()
    assert e.value.name == "DeviceTimeout"


# one tile a CTA and several of them, so that warps which have given up pass the barriers of tiles that others still read
@pytest.mark.parametrize("rows,k,n,off", [
    (60, 512, 3000, 0), (64, 2048, 19100, 0),               # 64 columns
    (130, 320, 9001, 0), (38000, 64, 128, 0),               # 128
    (700, 144, 6200, 0),                                    # 256
    (1000, 512, 4096, 0), (8192, 256, 4096, 0),             # pairs of CTAs
    (260, 511, 129, 1), (2000, 300, 2000, 3)])              # rows read where they are
@pytest.mark.parametrize("cta", [0, 1, 73, 1000001])
def test_a_cta_gives_up(zb, tight, rows, k, n, off, cta):
    import torch
    ops = operands(np.random.default_rng(rows), rows, k, n)
    pad = 0 if off else -k % 16
    tight.selftest_give_up(cta)
    timed_out(zb, lambda: product(tight, torch, *ops, "bf16", (off, pad), (off, pad)))
    for _ in range(2):
        sampled(torch, product(tight, torch, *ops, "bf16", (off, pad), (off, pad)), ops, "bf16")


@pytest.mark.parametrize("counts,k,n", [([40, 0, 129, 1, 260], 320, 2000), ([900, 1131, 2000], 256, 4096)])
def test_a_cta_of_a_grouped_product_gives_up(zb, tight, counts, k, n):
    import torch
    offsets = np.concatenate([[1], 1 + np.cumsum(counts)])
    ops = operands(np.random.default_rng(k), int(offsets[-1]) + 3, k, n, len(counts), bias=True)
    for cta in (0, 5):
        tight.selftest_give_up(cta)
        timed_out(zb, lambda: grouped(tight, torch, ops, offsets, "f16"))
    y = grouped(tight, torch, ops, offsets, "f16")
    r = np.r_[0:4, offsets[-1]:len(ops[0])]
    assert (y[torch.from_numpy(np.r_[0, offsets[-1]:len(ops[0])]).cuda()] == 77).all() and not (y[torch.from_numpy(r[1:4]).cuda()] == 77).all(dim=1).any()
    if k == 320:
        check_groups(y, ops, offsets, "f16")


def test_few_token_products_have_no_such_wait(zb, tight):
    """The self test stays armed over a kernel without bounded waits, and a negative CTA disarms it."""
    import torch
    ops = operands(np.random.default_rng(3), 3, 256, 100)
    tight.selftest_give_up(0)
    sampled(torch, product(tight, torch, *ops, "f32"), ops, "f32")
    tight.selftest_give_up(-1)
    ops = operands(np.random.default_rng(4), 300, 256, 4000)
    sampled(torch, product(tight, torch, *ops, "f32"), ops, "f32")


def test_kernels_close_behind_each_other(zb):
    """Short products of each kernel follow each other without a pause, on barriers at the same shared memory: none is disturbed by what the one before it
    has still under way, and none waits for long."""
    import torch
    c = zb.Context(0)
    stream = torch.cuda.Stream()
    c.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(11)
    work = []
    # pairs of CTAs before and behind each other kernel; k of one stage, of a few, of more than the ring holds
    for rows, k, n in ((1000, 512, 4096), (60, 128, 3000), (1000, 128, 4096), (130, 320, 9001), (8192, 144, 512), (700, 144, 6200), (1000, 1040, 4096), (5, 256, 128)):
        ops = operands(rng, rows, k, n)
        dev = [torch.from_numpy(v).cuda() for v in ops[:4]]
        want = (dev[0].double() @ dev[2].double().T).float() * dev[1][:, None] * dev[3]         # (exact sums, and the kernels' order of roundings)
        work.append((dev, torch.empty(rows, n, device="cuda"), want))
    torch.cuda.synchronize()
    for turn in range(40):
        for i in range(len(work)):
            dev, y, _ = work[(i * (1 + 2 * (turn % 4))) % len(work)]
            c.qmatmul_scaled(*dev, out=y)
        if turn % 8 == 7:
            c.synchronize()
            for _, y, want in work:
                assert torch.equal(y, want)
                y.fill_(77.0)
            torch.cuda.synchronize()
    c.set_stream(torch.cuda.default_stream().cuda_stream)
    c.close()
