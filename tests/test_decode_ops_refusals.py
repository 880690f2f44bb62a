"""Refusals of the operators on a decoder's int8 cache and of verify_drafts, and calls that have nothing to do: no GPU needed."""
import ctypes as C

import numpy as np
import pytest

F, I = np.float32, np.int32


@pytest.fixture(scope="module")
def nogpu(zb):
    return zb.Context(None)


def refused(zb, name, call):
    with pytest.raises(zb.ZantError) as e:
        call()
    assert e.value.name == name, e.value


def arrays(pages=4, heads=2, page=16, dim=32):
    return np.zeros((pages, heads, page, dim), np.int8), np.ones((pages, heads), F), np.zeros((pages, heads, page, dim), np.int8), np.ones((pages, heads), F)


def make(zb, **kw):
    return zb.KvCache(*arrays(**kw))


def ro(v):
    v.flags.writeable = False
    return v


def test_the_cache(zb):
    k, ks, v, vs = arrays()
    refused(zb, "InvalidRank", lambda: zb.KvCache(k[0], ks, v[0], vs))
    refused(zb, "InputTensorsWrongShape", lambda: zb.KvCache(k, ks, v[:2], vs))
    refused(zb, "InputArrayWrongSize", lambda: zb.KvCache(k, ks[:2], v, vs))
    refused(zb, "InputArrayWrongType", lambda: zb.KvCache(k.astype(np.uint8), ks, v, vs))
    refused(zb, "InputArrayWrongType", lambda: zb.KvCache(k, ks.astype(np.float16), v, vs))
    refused(zb, "InputArrayWrongType", lambda: zb.KvCache(k[:, :, ::2], ks, v[:, :, ::2], vs))
    refused(zb, "InputArrayWrongType", lambda: zb.KvCache(ro(arrays()[0]), ks, v, vs))
    import torch
    t = torch.zeros(4, 2, 16, 32, dtype=torch.int8)
    refused(zb, "WrongStride", lambda: zb.KvCache(torch.zeros(4, 16, 2, 32, dtype=torch.int8).transpose(1, 2), torch.ones(4, 2), t, torch.ones(4, 2)))
    refused(zb, "InputArrayWrongType", lambda: zb.KvCache(t.to(torch.uint8), torch.ones(4, 2), t, torch.ones(4, 2)))


@pytest.mark.parametrize("name", ["write", "read", "attend"])
def test_sizes(zb, nogpu, name):
    table, lengths = np.zeros((2, 2), I), np.array([20, 5], I)
    x = lambda rows=4, wide=64, t=F: np.zeros((rows, wide), t)  # noqa: E731

    def call(cache=None, a=None, b=None, table=table, lengths=lengths, offsets=None, **kw):
        cache = cache or make(zb)
        a = x() if a is None else a
        b = a if b is None else b
        if name == "write":
            return nogpu.kv_cache_write(cache, a, b, table, lengths, offsets=offsets)
        if name == "read":
            return nogpu.kv_cache_read(cache, table, lengths, offsets=offsets, out=(a, b))
        return nogpu.kv_cache_attention(cache, a, table, lengths, offsets=offsets, out=b, **kw)
    small = "OutputTensorDifferentSize" if name != "write" else "InputTensorsWrongShape"
    refused(zb, "CudaUnavailable", call)
    refused(zb, "CudaUnavailable", lambda: call(offsets=[0, 1, 4]))
    refused(zb, "CudaUnavailable", lambda: call(a=x(t=np.float16)))
    refused(zb, "CudaUnavailable", lambda: call(a=np.zeros((4, 2, 32), F)))
    refused(zb, "InputTensorDifferentSize", lambda: call(a=x(3)))
    refused(zb, "CudaUnavailable", lambda: call(a=x(3), offsets=[0, 1, 2]))
    refused(zb, small, lambda: call(b=x(5)))
    refused(zb, small, lambda: call(a=x(4, 64), b=x(4, 32)))
    refused(zb, "InputArrayWrongType", lambda: call(a=x(t=np.float64)))
    refused(zb, "InputArrayWrongType", lambda: call(b=x(t=np.float16)))
    refused(zb, "InvalidRank", lambda: call(a=np.zeros(64, F)))
    refused(zb, "InvalidRank", lambda: call(table=np.zeros(4, I)))
    refused(zb, "InputArrayWrongSize", lambda: call(lengths=[1, 2, 3]))
    refused(zb, "InputArrayWrongSize", lambda: call(offsets=[0, 4]))
    refused(zb, "InputArrayWrongType", lambda: call(table=np.zeros((2, 2))))
    refused(zb, "InputArrayWrongType", lambda: call(lengths=[1.0, 2.0]))
    for page in (8, 48, 512):
        refused(zb, "InvalidInput", lambda: call(cache=make(zb, page=page)))
    for dim in (8, 24, 272):
        refused(zb, "UnsupportedDimension", lambda: call(cache=make(zb, dim=dim), a=x(4, 2 * dim)))
    refused(zb, "InputTensorsWrongShape", lambda: call(cache=make(zb, pages=0)))
    # nothing to do
    call(a=x(0))
    call(a=x(0), table=np.zeros((0, 2), I), lengths=[])
    call(table=np.zeros((0, 2), I), lengths=[], offsets=[0])
    if name == "read":
        assert nogpu.kv_cache_read(make(zb), table, lengths, out=(None, None)) == (None, None)
        refused(zb, "NullPointer", lambda: nogpu.kv_cache_read(make(zb), table, lengths))
        refused(zb, "InputArrayWrongType", lambda: call(b=ro(x())))
        refused(zb, "CudaUnavailable", lambda: nogpu.kv_cache_read(make(zb), table, lengths, out=(None, x())))
    if name == "attend":
        refused(zb, "CudaUnavailable", lambda: call(a=x(4, 192)))
        refused(zb, "InputTensorsWrongShape", lambda: call(a=x(4, 96)))            # 3 heads over 2
        refused(zb, "InputTensorsWrongShape", lambda: call(a=x(4, 72)))
        refused(zb, "InvalidInput", lambda: call(window=-1))
        refused(zb, "InvalidInput", lambda: call(window=3, sinks=-1))
        refused(zb, "InputArrayWrongSize", lambda: call(lse=np.zeros(7, F)))
        refused(zb, "InputArrayWrongType", lambda: call(lse=np.zeros((4, 2), np.float16)))
        refused(zb, "InputArrayWrongType", lambda: call(b=ro(x())))
        assert nogpu.kv_cache_attention(make(zb), x(0), table, lengths).shape == (0, 64)
    import torch
    t = torch.zeros(4, 128)
    refused(zb, "CudaUnavailable", lambda: call(a=t[:, 64:], b=t[:, :64]))
    refused(zb, "CudaUnavailable", lambda: call(a=t.view(4, 4, 32)[:, 1:3], b=t.view(4, 4, 32)[:, 2:]))
    refused(zb, "WrongStride", lambda: call(a=t[:, ::2]))
    refused(zb, "WrongStride", lambda: call(a=t.view(4, 4, 32)[:, ::2]))
    refused(zb, "InputArrayWrongType", lambda: call(a=t[:, :64].to(torch.int8)))
    refused(zb, "InputArrayWrongType", lambda: call(table=torch.zeros(2, 2, dtype=torch.int64)))
    refused(zb, "WrongStride", lambda: call(table=torch.zeros(2, 4, dtype=torch.int32)[:, :2]))


def test_drafts(zb, nogpu):
    p, q, t, a, s = np.ones((8, 10), F), np.ones((6, 10), F), np.zeros(6, I), np.zeros(6, F), np.zeros(2, F)
    refused(zb, "CudaUnavailable", lambda: nogpu.verify_drafts(p, q, t, a, s))
    refused(zb, "CudaUnavailable", lambda: nogpu.verify_drafts(p, None, t, a, s, offsets=[0, 2, 6]))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.verify_drafts(p[:7], q, t, a, s))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.verify_drafts(p, q[:5], t, a, s))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.verify_drafts(p, q[:, :9], t, a, s))
    refused(zb, "InputArrayWrongType", lambda: nogpu.verify_drafts(p, q.astype(np.float16), t, a, s))
    refused(zb, "InputArrayWrongType", lambda: nogpu.verify_drafts(p.astype(np.float64), q.astype(np.float64), t, a, s))
    refused(zb, "InputArrayWrongType", lambda: nogpu.verify_drafts(p, q, t.astype(F), a, s))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.verify_drafts(p, q, t, a[:5], s))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.verify_drafts(p, q, t, a, s, offsets=[0, 6]))
    refused(zb, "InputTensorDifferentSize", lambda: nogpu.verify_drafts(np.ones((10, 10), F), q, t, a, np.zeros(4, F)))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.verify_drafts(np.ones((8, 0), F), None, t, a, s))
    refused(zb, "InputArrayWrongType", lambda: nogpu.verify_drafts(p, q, t, a, s, out=(np.zeros(2, I), ro(np.zeros(2, I)))))
    refused(zb, "InputArrayWrongType", lambda: nogpu.verify_drafts(p, q, t, a, s, out=(np.zeros(2, np.int64), np.zeros(2, I))))
    refused(zb, "CudaUnavailable", lambda: nogpu.verify_drafts(p[:2], None, t[:0], a[:0], s))
    n, f = nogpu.verify_drafts(p[:0], None, t[:0], a[:0], s[:0])
    assert n.shape == f.shape == (0,)


def test_c_entries(zb):
    """What the binding cannot pass: NULL, strides shorter than a row, counts beyond what the kernels hold."""
    L, z = zb.lib(), np.zeros(64, F)
    p = z.__array_interface__["data"][0]

    def name(status):
        return L.zant_b200_status_name(C.c_int32(status)).decode()

    def struct(k=p, ks=p, v=p, vs=p, pages=2, heads=2, page=16, dim=16):
        st = type(make(zb)._struct)(k, ks, v, vs, pages, heads, page, dim)
        struct.kept = st
        return C.addressof(st)

    def write(c=None, dtype=0, k=p, ks=0, v=p, vs=0, rows=2, table=p, seqs=2, width=1, lengths=p, offsets=None):
        return name(L.zant_b200_kv_cache_write(None, struct() if c is None else c, dtype, k, ks, v, vs, rows, table, seqs, width, lengths, offsets))

    def read(c=None, dtype=0, k=p, ks=0, v=p, vs=0, rows=2, table=p, seqs=2, width=1, lengths=p, offsets=None):
        return name(L.zant_b200_kv_cache_read(None, struct() if c is None else c, dtype, k, ks, v, vs, rows, table, seqs, width, lengths, offsets))

    def attend(c=None, dtype=0, k=p, ks=0, v=p, vs=0, rows=2, table=p, seqs=2, width=1, lengths=p, offsets=None, heads=4, window=0, sinks=0):
        return name(L.zant_b200_kv_cache_attention(None, struct() if c is None else c, dtype, k, ks, rows, heads, table, seqs, width, lengths, offsets, 1.0, window, sinks, v, vs, None))
    for f in (write, read, attend):
        assert f() == f(dtype=4) == f(dtype=5) == f(offsets=p) == f(width=0, table=None) == "CudaUnavailable"
        assert f(dtype=1) == f(dtype=6) == "InputArrayWrongType"
        assert f(c=0) == f(table=None) == f(lengths=None) == f(c=struct(k=None)) == f(c=struct(vs=None)) == "NullPointer"
        if f is not read:
            assert f(k=None) == f(v=None) == "NullPointer"
        assert f(ks=31) == f(vs=31) == "WrongStride"
        assert f(c=struct(heads=0)) == f(c=struct(pages=0)) == "InputTensorsWrongShape"
        assert f(c=struct(page=24)) == f(c=struct(page=0)) == f(c=struct(page=1 << 40)) == "InvalidInput"
        assert f(c=struct(dim=0)) == f(c=struct(dim=40)) == f(c=struct(dim=1 << 40)) == "UnsupportedDimension"
        assert f(rows=1 << 31) == f(width=1 << 31) == f(seqs=1 << 25, rows=0) == f(ks=1 << 62) == f(c=struct(pages=1 << 31)) == "TooLarge"
        assert f(seqs=0) == f(rows=3) == "InputTensorDifferentSize"
        assert f(rows=0, k=None, v=None, lengths=None) == f(seqs=0, offsets=p) == "OK"
    assert write(c=struct(heads=65536)) == read(c=struct(heads=65536)) == "TooLarge"
    assert attend(heads=3) == attend(heads=0) == "InputTensorsWrongShape" and attend(heads=65536) == "TooLarge"
    assert attend(window=-1) == attend(sinks=-5) == "InvalidInput"

    def verify(dtype=0, t=p, ts=0, d=p, ds=0, vocab=4, tokens=p, drafts=2, offsets=None, seqs=2, accept=p, sample=p, n=p, nxt=p):
        return name(L.zant_b200_verify_drafts(None, dtype, t, ts, d, ds, vocab, tokens, drafts, offsets, seqs, accept, sample, n, nxt))
    assert verify() == verify(d=None) == verify(drafts=0, tokens=None, accept=None) == verify(drafts=3, offsets=p) == "CudaUnavailable"
    assert verify(t=None) == verify(tokens=None) == verify(accept=None) == verify(sample=None) == verify(n=None) == verify(nxt=None) == "NullPointer"
    assert verify(ts=3) == verify(ds=3) == "WrongStride" and verify(dtype=3) == "InputArrayWrongType" and verify(vocab=0) == "InputTensorsWrongShape"
    assert verify(drafts=3) == "InputTensorDifferentSize"
    assert verify(vocab=1 << 31) == verify(drafts=1 << 31) == verify(seqs=1 << 25) == verify(ts=1 << 62) == "TooLarge"
    assert verify(seqs=0, drafts=0, t=None) == "OK"
