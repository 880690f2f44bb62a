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
