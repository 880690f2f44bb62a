"""quantize_rows against exact quotients in 64 bits: codes and scales are equal bit for bit."""
import numpy as np
import pytest

import token_ops_reference as ref

pytestmark = pytest.mark.gpu
TYPES = ("f32", "f16", "bf16")


def torch_type(torch, t):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def check(q, s, x, index=None):
    """q, s: device results; x: the device tensor they were made from."""
    want_q, want_s = ref.quantize_rows(x.double().cpu().numpy(), index)
    got_s = s.cpu().numpy()
    assert np.array_equal(got_s, want_s, equal_nan=True), (got_s, want_s)
    bad = np.argwhere(q.cpu().numpy() != want_q)
    assert not len(bad), (len(bad), bad[:5])


def run(ctx, torch, x, index=None, pad=0):
    rows = x.shape[0] if index is None else len(index)
    room = torch.full((rows, x.shape[1] + pad), 77, dtype=torch.int8, device="cuda")
    q, s = room[:, :x.shape[1]], torch.full((rows,), 5.0, device="cuda")
    torch.cuda.synchronize()
    got = ctx.quantize_rows(x, index=None if index is None else torch.from_numpy(index).cuda(), out=q, out_scale=s)
    ctx.synchronize()
    assert got[0] is q and got[1] is s
    assert (room[:, x.shape[1]:] == 77).all()
    return q, s


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 7, 16, 33, 128, 255, 1000, 1024, 2049, 4096, 4099, 8192, 16384, 20011, 40000])
def test_sizes(ctx, t, cols):
    import torch
    g = torch.Generator(device="cuda").manual_seed(cols)
    for rows in (1, 5, 300):
        x = (torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))).to(torch_type(torch, t))
        check(*run(ctx, torch, x), x)


@pytest.mark.parametrize("t", TYPES)
def test_special_rows(ctx, t):
    import torch
    d = torch_type(torch, t)
    fi = torch.finfo(d)
    cols = 50
    r = torch.linspace(-1, 1, cols, device="cuda")
    rows = [r * 0, r * -0.0, r * fi.max, r * fi.tiny, r * fi.smallest_normal * 130, r * float(fi.tiny) * 2.0 ** -4, torch.full_like(r, float(fi.max)), r * 1e-20, r * 127,
            torch.arange(cols, device="cuda") - 20.5, torch.cat([torch.arange(cols - 1, device="cuda") + 0.5, torch.tensor([127.0], device="cuda")])]
    for bad in (float("nan"), float("inf"), -float("inf")):
        v = r.clone()
        v[17] = bad
        rows.append(v)
    x = torch.stack(rows).to(d)
    x[0, 3] = 0.0
    check(*run(ctx, torch, x), x)
    # ties: with a largest value of 127 the scale is 1
    h = torch.arange(-254, 255, device="cuda") / 2
    x = h.to(d)[None]
    q, s = run(ctx, torch, x)
    assert s.item() == 1.0 and torch.equal(q[0].float(), torch.round(h).float())


def test_smallest_numbers(ctx):
    """Rows of subnormal numbers: the scale is rounded coarsely, codes saturate, or the scale vanishes."""
    import torch
    n = torch.tensor([[1, 0, 1], [60, 3, -60], [64, 1, -5], [100, -100, 50], [190, 95, -190], [191, -64, 32], [200, 100, -100], [2 ** 20, 12345, -2 ** 19], [2 ** 23, 2 ** 22, 99]], device="cuda")
    x = (n.double() * 2.0 ** -149).float()
    assert (x != 0).any()
    check(*run(ctx, torch, x), x)


@pytest.mark.parametrize("t", TYPES)
def test_near_ties(ctx, t):
    """Values one step of their type to either side of a border between two codes."""
    import torch
    rng = np.random.default_rng(3)
    d = torch_type(torch, t)
    top = torch.from_numpy(np.exp(rng.uniform(-3, 3, 64))).to(d).double()
    scale = (top / 127).float().double()
    border = (torch.arange(127).double() + 0.5)[None] * scale[:, None]
    x = border.to(d)
    step = torch.finfo(d).eps * x.double()
    cols = [top[:, None], x.double(), x.double() + step, x.double() - step]
    x = torch.cat(cols, 1)
    x = torch.minimum(x, top[:, None]).to(d).cuda()
    check(*run(ctx, torch, x), x)


@pytest.mark.parametrize("t", TYPES)
def test_index(ctx, t):
    import torch
    rng = np.random.default_rng(1)
    x = torch.randn(37, 515, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(torch_type(torch, t))
    index = rng.integers(0, 37, 200).astype(np.int32)
    index[[0, 7, 50]] = -1
    index[[1, 9]] = [37, 2 ** 31 - 1]
    index[10] = -2 ** 31
    check(*run(ctx, torch, x, index, pad=13), x, index)
    none = torch.empty(0, 515, device="cuda", dtype=x.dtype)
    q, s = run(ctx, torch, none, np.array([0, -1], np.int32))
    assert (q == 0).all() and (s == 0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", [64, 1001, 4096])
def test_strides_and_addresses(ctx, t, cols):
    """Rows apart, and tensors that begin at any element."""
    import torch
    room = torch.randn(9, cols + 40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(torch_type(torch, t))
    for off in (0, 1, 3, 8):
        x = room[:, off:off + cols]
        for pad in (0, 1, 16):
            check(*run(ctx, torch, x, pad=pad), x)
    flat = torch.full((5 * cols + 20,), 77, dtype=torch.int8, device="cuda")
    for off in (1, 2, 7):
        x, q, s = room[:5, :cols], flat[off:off + 5 * cols].view(5, cols), torch.empty(5, device="cuda")
        torch.cuda.synchronize()
        ctx.quantize_rows(x, out=q, out_scale=s)
        ctx.synchronize()
        check(q, s, x)
        assert (flat[:off] == 77).all() and (flat[off + 5 * cols:] == 77).all()
        flat.fill_(77)


def test_far_rows(ctx):
    """Rows whose offsets need more than 32 bits."""
    import torch
    base = torch.empty(2 ** 31 + 4096, dtype=torch.float16, device="cuda")
    x = base.as_strided((2, 1000), (2 ** 31 + 8, 1))
    x.copy_(torch.randn(2, 1000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)))
    check(*run(ctx, torch, x), x)
    qs = torch.empty(2 ** 31 + 4096, dtype=torch.int8, device="cuda").as_strided((2, 1000), (2 ** 31 + 8, 1))
    s = torch.empty(2, device="cuda")
    torch.cuda.synchronize()
    ctx.quantize_rows(x, out=qs, out_scale=s)
    ctx.synchronize()
    check(qs, s, x)


def test_host_arrays(ctx):
    rng = np.random.default_rng(5)
    for dt in (np.float32, np.float16):
        x = rng.standard_normal((11, 130)).astype(dt)
        index = np.array([3, 3, -1, 10, 0], np.int32)
        for ix in (None, index):
            q, s = ctx.quantize_rows(x, index=ix)
            wq, ws = ref.quantize_rows(x.astype(np.float64), ix)
            assert np.array_equal(q, wq) and np.array_equal(s, ws)


def test_equals_quantize_linear_away_from_ties(ctx):
    """With the row's scale QuantizeLinear gives the same codes; fp32 division rounds some quotients onto a tie (half a step in 2**17, twice)."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1, 4096)).astype(np.float32)
    q, s = ctx.quantize_rows(x)
    same = ctx.quantize_linear(x[0], float(s[0]), 0, out_dtype=1) == q[0]
    exact = np.abs(x[0].astype(np.float64) / s[0]) % 1
    assert same[np.abs(exact - 0.5) > 2.0 ** -17].all()


def test_misaligned_device_pointer_is_refused(zb, ctx):
    import ctypes as C
    import torch
    x, q, s = torch.zeros(64, device="cuda"), torch.zeros(64, dtype=torch.int8, device="cuda"), torch.zeros(8, device="cuda")
    L = zb.lib()
    for args in ((0, x.data_ptr() + 2, s.data_ptr()), (4, x.data_ptr() + 1, s.data_ptr()), (0, x.data_ptr(), s.data_ptr() + 1)):
        status = L.zant_b200_quantize_rows(ctx._h, args[0], args[1], 2, 8, 0, None, 2, q.data_ptr(), 0, args[2])
        assert L.zant_b200_status_name(C.c_int32(status)) == b"InvalidInput"
