"""qmatmul_scaled and qmatmul_grouped against 64-bit products."""
import numpy as np
import pytest

import token_ops_reference as ref

pytestmark = pytest.mark.gpu
TYPES = ("f32", "f16", "bf16")


def torch_type(torch, t):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def operands(rng, rows, k, n, groups=None, bias=False):
    a = rng.integers(-127, 128, (rows, k), dtype=np.int8)
    lead = () if groups is None else (groups,)
    w = rng.integers(-128, 128, lead + (n, k), dtype=np.int8)
    a_scale = np.exp(rng.uniform(-6, -2, rows)).astype(np.float32)
    w_scale = np.exp(rng.uniform(-6, -4, lead + (n,))).astype(np.float32)
    return a, a_scale, w, w_scale, rng.standard_normal(lead + (n,)).astype(np.float32) if bias else None


def place(torch, v, off=0, pad=0):
    """An int8 or float array on the device, its rows `pad` further apart than dense, its first element `off` elements into an allocation."""
    if v is None:
        return None
    v = torch.from_numpy(v)
    shape = v.shape
    row = shape[-1] + pad
    flat = torch.zeros(off + int(np.prod(shape[:-1])) * row, dtype=v.dtype, device="cuda")
    strides = [row, 1] if len(shape) == 2 else [shape[1] * row, row, 1]
    out = flat[off:].as_strided(shape, strides[-len(shape):])
    out.copy_(v)
    return out


def check(got, a, a_scale, w, w_scale, bias, t):
    want, off = ref.scaled_product(a, a_scale, w, w_scale, bias, t)
    d = np.abs(got.double().cpu().numpy() - want)
    assert (d <= off).all(), (float((d / off).max()), np.argwhere(d > off)[:4])


def product(ctx, torch, a, a_scale, w, w_scale, bias, t, a_at=(0, 0), w_at=(0, 0), y_at=(0, 0)):
    rows, n = a.shape[0], w.shape[0]
    room = torch.full((y_at[0] + rows * (n + y_at[1]),), 77.0, dtype=torch_type(torch, t), device="cuda")
    y = room[y_at[0]:].as_strided((rows, n), (n + y_at[1], 1))
    args = place(torch, a, *a_at), torch.from_numpy(a_scale).cuda(), place(torch, w, *w_at), torch.from_numpy(w_scale).cuda()
    b = None if bias is None else torch.from_numpy(bias).cuda()
    torch.cuda.synchronize()
    assert ctx.qmatmul_scaled(*args, bias=b, out=y) is y
    ctx.synchronize()
    mask = torch.ones_like(room, dtype=torch.bool)
    mask[y_at[0]:].as_strided((rows, n), (n + y_at[1], 1)).fill_(False)
    assert (room[mask] == 77.0).all(), "wrote beside its rows"
    return y


ROWS = [1, 2, 3, 15, 16, 17, 31, 33, 64, 65, 100, 127, 129, 256, 257, 300, 513]


@pytest.mark.parametrize("rows", ROWS)
def test_rows(ctx, rows):
    import torch
    rng = np.random.default_rng(rows)
    for i, (k, n) in enumerate(((256, 384), (1040, 130), (4096, 640))):
        ops = operands(rng, rows, k, n, bias=i == 1)
        check(product(ctx, torch, *ops, TYPES[(rows + i) % 3]), *ops, TYPES[(rows + i) % 3])


@pytest.mark.parametrize("k", [1, 2, 15, 16, 17, 31, 32, 33, 48, 100, 127, 128, 129, 144, 255, 256, 272, 1000, 1001, 2064, 4095, 9999])
def test_depths(ctx, k):
    import torch
    rng = np.random.default_rng(k)
    for i, (rows, n) in enumerate(((1, 200), (20, 65), (150, 129))):
        ops = operands(rng, rows, k, n)
        check(product(ctx, torch, *ops, TYPES[i]), *ops, TYPES[i])


@pytest.mark.parametrize("n", [1, 2, 3, 8, 31, 32, 63, 64, 65, 127, 128, 129, 200, 256, 257, 1000, 2000, 5001])
def test_widths(ctx, n):
    import torch
    rng = np.random.default_rng(n)
    for i, (rows, k) in enumerate(((1, 512), (40, 304), (260, 128))):
        ops = operands(rng, rows, k, n, bias=True)
        check(product(ctx, torch, *ops, TYPES[(i + n) % 3]), *ops, TYPES[(i + n) % 3])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("a_at,w_at,y_at", [((0, 16), (0, 32), (0, 5)), ((1, 0), (0, 0), (0, 0)), ((0, 0), (3, 0), (1, 0)), ((0, 1), (0, 0), (0, 8)), ((0, 0), (0, 7), (3, 3)), ((16, 112), (48, 16), (8, 24))])
def test_addresses(ctx, t, a_at, w_at, y_at):
    import torch
    rng = np.random.default_rng(8)
    for rows, k, n in ((1, 512, 256), (33, 640, 300), (200, 256, 129)):
        ops = operands(rng, rows, k, n, bias=True)
        check(product(ctx, torch, *ops, t, a_at, w_at, y_at), *ops, t)


@pytest.mark.parametrize("rows,k,n", [(1024, 1024, 1024), (2050, 3000, 1111), (777, 4112, 4097), (4096, 512, 2048), (8, 16384, 8200), (64, 14336, 4096), (130, 8192, 8192)])
def test_large(ctx, rows, k, n):
    import torch
    rng = np.random.default_rng(k)
    ops = operands(rng, rows, k, n, bias=True)
    t = TYPES[rows % 3]
    y = product(ctx, torch, *ops, t)
    # 64-bit products of all of it take too long on the host: rows and columns of every part
    r = np.unique(np.concatenate([np.arange(min(rows, 8)), rng.integers(0, rows, 60), np.arange(max(0, rows - 8), rows)]))
    c = np.unique(np.concatenate([np.arange(8), rng.integers(0, n, 200), np.arange(n - 8, n)]))
    check(y[torch.from_numpy(r).cuda()][:, torch.from_numpy(c).cuda()], ops[0][r], ops[1][r], ops[2][c], ops[3][c], ops[4][c], t)
    exact = torch.from_numpy(ops[0]).cuda().double() @ torch.from_numpy(ops[2]).cuda().double().T
    want = exact * torch.from_numpy(ops[1]).cuda().double()[:, None] * torch.from_numpy(ops[3]).cuda().double() + torch.from_numpy(ops[4]).cuda().double()
    off = (4.1 * ref.U + ref.HALF_STEP[t] * 1.01) * (want.abs() + torch.from_numpy(np.abs(ops[4])).cuda().double()) * 2 + 1e-30
    assert ((y.double() - want).abs() <= off).all()


def test_largest_sums(ctx):
    """131071 products of -128 and -128 are 16384 below the end of int32; sums of one sign at every kernel's depth."""
    import torch
    for rows, k, n in ((2, 131071, 3), (2, 131056, 130), (40, 131056, 64)):
        a, w = np.full((rows, k), -128, np.int8), np.full((n, k), -128, np.int8)
        w[1] = 127
        one = np.ones(rows, np.float32), np.ones(n, np.float32)
        check(product(ctx, torch, a, one[0], w, one[1], None, "f32"), a, one[0], w, one[1], None, "f32")


def test_scales_of_any_kind(ctx):
    """Zero, negative, infinite and NaN scales stay in their row or column; f16 results overflow to infinity."""
    import torch
    rng = np.random.default_rng(9)
    a, a_scale, w, w_scale, _ = operands(rng, 20, 64, 40)
    a_scale[[0, 3, 5]] = [0, np.nan, -1]
    w_scale[[2, 7]] = [np.nan, 1e30]
    for t in TYPES:
        y = product(ctx, torch, a, a_scale, w, w_scale, None, t).double().cpu().numpy()
        with np.errstate(all="ignore"):
            want, off = ref.scaled_product(a, a_scale, w, w_scale, None, t)
        assert np.isnan(y[3]).all() and np.isnan(y[:, 2]).all()
        fine = np.isfinite(want)
        if t == "f16":
            big = fine & (np.abs(want) > 65520)
            assert big.any() and np.array_equal(y[big], np.sign(want[big]) * np.inf)
            fine &= ~big
        assert (np.abs(y - want)[fine] <= off[fine]).all()


def test_far_operands(ctx):
    """Rows of either operand and of the result whose offsets need more than 32 bits."""
    import torch
    rng = np.random.default_rng(10)
    a, a_scale, w, w_scale, _ = operands(rng, 2, 320, 2)
    dev = [torch.from_numpy(v).cuda() for v in (a_scale, w_scale)]
    far = 2 ** 31 + 16
    for step in (far, far + 1):          # one is taken by the tensor memory accelerator, one is not
        A = torch.zeros(step + 320, dtype=torch.int8, device="cuda").as_strided((2, 320), (step, 1))
        W = torch.zeros(step + 320, dtype=torch.int8, device="cuda").as_strided((2, 320), (step, 1))
        Y = torch.zeros(step + 320, dtype=torch.float16, device="cuda").as_strided((2, 2), (step, 1))
        A.copy_(torch.from_numpy(a)); W.copy_(torch.from_numpy(w))
        torch.cuda.synchronize()
        ctx.qmatmul_scaled(A, dev[0], W, dev[1], out=Y)
        ctx.synchronize()
        check(Y, a, a_scale, w, w_scale, None, "f16")
        del A, W, Y


def grouped(ctx, torch, ops, offsets, t, y_pad=0, a_at=(0, 0), w_at=(0, 0)):
    a, a_scale, w, w_scale, bias = ops
    rows, n = a.shape[0], w.shape[1]
    room = torch.full((rows, n + y_pad), 77.0, dtype=torch_type(torch, t), device="cuda")
    y = room[:, :n]
    dev = place(torch, a, *a_at), torch.from_numpy(a_scale).cuda(), place(torch, w, *w_at), torch.from_numpy(w_scale).cuda(), torch.from_numpy(np.asarray(offsets, np.int32)).cuda()
    b = None if bias is None else torch.from_numpy(bias).cuda()
    torch.cuda.synchronize()
    assert ctx.qmatmul_grouped(*dev, bias=b, out=y) is y
    ctx.synchronize()
    assert (room[:, n:] == 77.0).all()
    return y


def check_groups(y, ops, offsets, t):
    a, a_scale, w, w_scale, bias = ops
    taken = np.zeros(len(a), bool)
    for g in range(len(offsets) - 1):
        b, e = offsets[g], offsets[g + 1]
        if e > b:
            check(y[b:e], a[b:e], a_scale[b:e], w[g], w_scale[g], None if bias is None else bias[g], t)
            taken[b:e] = True
    assert (y.float().cpu().numpy()[~taken] == 77.0).all(), "rows of no group were written"


COUNTS = [[5], [0, 0, 7], [1, 1, 1, 1], [16, 0, 17, 200, 1], [0, 300, 0], [64, 128, 256, 31], [3] * 64, [0] * 20 + [40] + [0] * 20, [130, 2, 0, 0, 90, 257]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("k,n", [(128, 128), (320, 200), (1000, 65), (77, 31), (1024, 512)])
def test_groups(ctx, counts, k, n):
    import torch
    rng = np.random.default_rng(k + len(counts))
    spare = 9 if len(counts) % 2 else 0
    offsets = np.concatenate([[0], np.cumsum(counts)])
    ops = operands(rng, sum(counts) + spare, k, n, len(counts), bias=k == 320)
    t = TYPES[(k + len(counts)) % 3]
    check_groups(grouped(ctx, torch, ops, offsets, t, y_pad=n % 3), ops, offsets, t)


def test_group_offsets_that_start_late_or_leave_gaps(ctx):
    import torch
    rng = np.random.default_rng(11)
    ops = operands(rng, 60, 256, 96, 3)
    offsets = [10, 20, 20, 47]
    check_groups(grouped(ctx, torch, ops, offsets, "f32"), ops, offsets, "f32")


@pytest.mark.parametrize("offsets", [[-5, 10, 30, 99], [30, 10, 40, 20], [2 ** 31 - 1, -2 ** 31, 7, 2 ** 31 - 1], [60, 60, 60, 60], [100, 200, 300, 400], [-4, -3, -2, -1]])
def test_broken_offsets_stay_inside(ctx, offsets):
    """Offsets are taken as clamped and as the largest so far."""
    import torch
    rng = np.random.default_rng(12)
    ops = operands(rng, 60, 256, 96, 3)
    y = grouped(ctx, torch, ops, offsets, "f32")
    check_groups(y, ops, np.maximum.accumulate(np.clip(np.asarray(offsets, np.int64), 0, 60)), "f32")


def test_many_groups(ctx):
    import torch
    rng = np.random.default_rng(13)
    counts = rng.integers(0, 4, 1024)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    ops = operands(rng, int(offsets[-1]), 144, 40, 1024)
    check_groups(grouped(ctx, torch, ops, offsets, "bf16"), ops, offsets, "bf16")


@pytest.mark.parametrize("a_at,w_at", [((0, 16), (16, 16)), ((1, 0), (0, 0)), ((0, 0), (5, 0)), ((0, 3), (0, 3))])
def test_group_addresses(ctx, a_at, w_at):
    import torch
    rng = np.random.default_rng(14)
    offsets = [0, 33, 40, 40, 170]
    ops = operands(rng, 175, 272, 150, 4, bias=True)
    check_groups(grouped(ctx, torch, ops, offsets, "f16", 2, a_at, w_at), ops, offsets, "f16")


def test_host_arrays(ctx):
    rng = np.random.default_rng(15)
    for k in (64, 75):
        ops = operands(rng, 9, k, 21, bias=True)
        want, off = ref.scaled_product(*ops, "f32")
        assert (np.abs(ctx.qmatmul_scaled(*ops) - want) <= off).all()
        ops = operands(rng, 9, k, 21, 3)
        out = np.full((9, 21), 77, np.float16)
        assert ctx.qmatmul_grouped(*ops[:4], [1, 4, 4, 8], out=out) is out
        assert (out[[0, 8]] == 77).all()
        for b, e, g in ((1, 4, 0), (4, 8, 2)):
            want, off = ref.scaled_product(ops[0][b:e], ops[1][b:e], ops[2][g], ops[3][g], None, "f16")
            assert (np.abs(out[b:e].astype(np.float64) - want) <= off).all()


def test_same_sums_at_any_address(ctx):
    """Exact sums: operands that the tensor memory accelerator reads and ones that it cannot give the same bits."""
    import torch
    rng = np.random.default_rng(16)
    for rows in (1, 70, 300):
        ops = operands(rng, rows, 2048, 600, bias=True)
        y = [product(ctx, torch, *ops, "f32", a_at, w_at) for a_at, w_at in (((0, 0), (0, 0)), ((0, 1), (0, 0)), ((0, 0), (1, 0)))]
        assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
