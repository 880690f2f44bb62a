"""Refusals of quantize_rows, qmatmul_scaled, qmatmul_grouped and token_logprobs, and calls that have nothing to do: no GPU needed."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture(scope="module")
def nogpu(zb):
    return zb.Context(None)


def refused(zb, name, call):
    with pytest.raises(zb.ZantError) as e:
        call()
    assert e.value.name == name, e.value


F = np.float32


def test_quantize_rows(zb, nogpu):
    x = np.ones((3, 8), F)
    refused(zb, "CudaUnavailable", lambda: nogpu.quantize_rows(x))
    refused(zb, "CudaUnavailable", lambda: nogpu.quantize_rows(x, index=[0, 2, -1, 7]))
    refused(zb, "InvalidRank", lambda: nogpu.quantize_rows(np.ones(8, F)))
    refused(zb, "InputArrayWrongType", lambda: nogpu.quantize_rows(np.ones((3, 8), np.float64)))
    refused(zb, "InputArrayWrongType", lambda: nogpu.quantize_rows(np.ones((3, 8), np.int8)))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.quantize_rows(np.ones((3, 0), F)))
    refused(zb, "OutputTensorDifferentSize", lambda: nogpu.quantize_rows(x, out=np.zeros((3, 7), np.int8)))
    refused(zb, "InputArrayWrongType", lambda: nogpu.quantize_rows(x, out=np.zeros((3, 8), np.int32)))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.quantize_rows(x, out_scale=np.zeros(4, F)))
    refused(zb, "InputArrayWrongType", lambda: nogpu.quantize_rows(x, out_scale=np.zeros(3, np.float16)))
    q, s = nogpu.quantize_rows(np.ones((0, 8), F))
    assert q.shape == (0, 8) and s.shape == (0,)


def test_torch_strides(zb, nogpu):
    import torch
    x = torch.ones(6, 16)
    refused(zb, "CudaUnavailable", lambda: nogpu.quantize_rows(x[::2, :7]))
    refused(zb, "WrongStride", lambda: nogpu.quantize_rows(x[:, ::2]))
    refused(zb, "WrongStride", lambda: nogpu.quantize_rows(x[:1].expand(4, 16)))
    refused(zb, "WrongStride", lambda: nogpu.quantize_rows(x.t()))
    refused(zb, "InputArrayWrongType", lambda: nogpu.quantize_rows(x, index=torch.zeros(2, dtype=torch.int64)))
    refused(zb, "WrongStride", lambda: nogpu.quantize_rows(x, out_scale=torch.ones(12)[::2]))
    w = torch.ones(4, 10, 16, dtype=torch.int8)
    a, s = torch.ones(6, 16, dtype=torch.int8), torch.ones(6)
    off = torch.zeros(3, dtype=torch.int32)
    refused(zb, "WrongStride", lambda: nogpu.qmatmul_grouped(a, s, w[::2], torch.ones(2, 10), off, out=torch.zeros(6, 10)))
    refused(zb, "WrongStride", lambda: nogpu.qmatmul_grouped(a, s, w[:2, :5], torch.ones(2, 5), off, out=torch.zeros(6, 5)))
    refused(zb, "CudaUnavailable", lambda: nogpu.qmatmul_grouped(a[:, :12], s, w[:2, :, :12], torch.ones(2, 10), off, out=torch.zeros(6, 10)))


def test_products(zb, nogpu):
    a, s, w, ws = np.ones((3, 8), np.int8), np.ones(3, F), np.ones((5, 8), np.int8), np.ones(5, F)
    refused(zb, "CudaUnavailable", lambda: nogpu.qmatmul_scaled(a, s, w, ws))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.qmatmul_scaled(a, s, np.ones((5, 9), np.int8), ws))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.qmatmul_scaled(a, s, np.ones((0, 8), np.int8), np.ones(0, F)))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.qmatmul_scaled(np.ones((3, 0), np.int8), s, np.ones((5, 0), np.int8), ws))
    refused(zb, "InputArrayWrongType", lambda: nogpu.qmatmul_scaled(a.astype(np.int32), s, w, ws))
    refused(zb, "InputArrayWrongType", lambda: nogpu.qmatmul_scaled(a, s, w.astype(np.uint8), ws))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.qmatmul_scaled(a, np.ones(4, F), w, ws))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.qmatmul_scaled(a, s, w, np.ones(1, F)))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.qmatmul_scaled(a, s, w, ws, bias=np.ones(6, F)))
    refused(zb, "InputArrayWrongType", lambda: nogpu.qmatmul_scaled(a, s, w, ws, y_dtype=zb.BF16))
    refused(zb, "InputArrayWrongType", lambda: nogpu.qmatmul_scaled(a, s, w, ws, y_dtype=zb.I8))
    refused(zb, "InputArrayWrongType", lambda: nogpu.qmatmul_scaled(a, s, w, ws, out=np.zeros((3, 5), np.int8)))
    refused(zb, "OutputTensorDifferentSize", lambda: nogpu.qmatmul_scaled(a, s, w, ws, out=np.zeros((3, 6), F)))
    k = 131072
    refused(zb, "TooLarge", lambda: nogpu.qmatmul_scaled(np.ones((1, k), np.int8), np.ones(1, F), np.ones((1, k), np.int8), np.ones(1, F)))
    refused(zb, "CudaUnavailable", lambda: nogpu.qmatmul_scaled(np.ones((1, k - 1), np.int8), np.ones(1, F), np.ones((1, k - 1), np.int8), np.ones(1, F)))
    assert nogpu.qmatmul_scaled(a[:0], s[:0], w, ws).shape == (0, 5)


def test_grouped(zb, nogpu):
    a, s, w, ws = np.ones((3, 8), np.int8), np.ones(3, F), np.ones((2, 5, 8), np.int8), np.ones((2, 5), F)
    refused(zb, "CudaUnavailable", lambda: nogpu.qmatmul_grouped(a, s, w, ws, [0, 1, 3]))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.qmatmul_grouped(a, s, w, ws, [0, 3]))
    refused(zb, "NullPointer", lambda: nogpu.qmatmul_grouped(a, s, w, ws, None))
    refused(zb, "InvalidRank", lambda: nogpu.qmatmul_grouped(a, s, w[0], ws[0], [0, 3]))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.qmatmul_grouped(a, s, w[:0], ws[:0], [0]))
    many = np.ones((1025, 1, 8), np.int8)
    refused(zb, "TooLarge", lambda: nogpu.qmatmul_grouped(a, s, many, np.ones((1025, 1), F), np.zeros(1026, np.int32)))


def test_logprobs(zb, nogpu):
    x = np.zeros((2, 10), F)
    refused(zb, "CudaUnavailable", lambda: nogpu.token_logprobs(x, [0, 1]))
    refused(zb, "CudaUnavailable", lambda: nogpu.token_logprobs(x, top=10))
    refused(zb, "InvalidInput", lambda: nogpu.token_logprobs(x, top=11))
    refused(zb, "InvalidInput", lambda: nogpu.token_logprobs(x, top=-1))
    refused(zb, "InvalidInput", lambda: nogpu.token_logprobs(np.zeros((2, 100), F), top=33))
    refused(zb, "InputArrayWrongSize", lambda: nogpu.token_logprobs(x, [0, 1, 2]))
    refused(zb, "InputArrayWrongType", lambda: nogpu.token_logprobs(x.astype(np.int8), [0, 1]))
    refused(zb, "InputTensorsWrongShape", lambda: nogpu.token_logprobs(np.zeros((2, 0), F), [0, 1]))
    out = (None, np.zeros(2, F), np.zeros((2, 0), np.int32), np.zeros((2, 0), F))
    refused(zb, "NullPointer", lambda: nogpu.token_logprobs(x, [0, 1], out=out))
    lp, h, ids, likely = nogpu.token_logprobs(x[:0], np.zeros(0, np.int32), top=3)
    assert lp.shape == h.shape == (0,) and ids.shape == likely.shape == (0, 3)


def test_c_entries(zb):
    """What the binding cannot pass: strides shorter than a row, spans beyond an address, NULL, other types."""
    L, z = zb.lib(), np.zeros(64, F)
    p = z.__array_interface__["data"][0]

    def name(status):
        return L.zant_b200_status_name(C.c_int32(status)).decode()

    def quant(dtype=0, x=p, rows=4, cols=8, stride=0, index=None, out_rows=4, q=p, q_stride=0, scale=p):
        return name(L.zant_b200_quantize_rows(None, dtype, x, rows, cols, stride, index, out_rows, q, q_stride, scale))
    assert quant() == "CudaUnavailable"
    assert quant(stride=7) == quant(q_stride=7) == "WrongStride"
    assert quant(dtype=1) == quant(dtype=6) == "InputArrayWrongType"
    assert quant(out_rows=3) == "InputTensorDifferentSize"
    assert quant(x=None) == quant(q=None) == quant(scale=None) == "NullPointer"
    assert quant(rows=1 << 31, out_rows=1 << 31) == quant(cols=1 << 31) == quant(stride=1 << 61) == "TooLarge"
    assert quant(rows=0, out_rows=0, x=None, q=None, scale=None) == "OK"
    assert quant(rows=0, x=None, index=p) == "CudaUnavailable"

    def product(a=p, rows=2, k=8, a_stride=0, a_scale=p, w=p, n=3, w_stride=0, w_scale=p, bias=None, y_dtype=0, y=p, y_stride=0):
        return name(L.zant_b200_qmatmul_scaled(None, a, rows, k, a_stride, a_scale, w, n, w_stride, w_scale, bias, y_dtype, y, y_stride))
    assert product() == product(y_dtype=5) == "CudaUnavailable"
    assert product(a_stride=7) == product(w_stride=1) == product(y_stride=2) == "WrongStride"
    assert product(y_dtype=3) == product(y_dtype=-1) == "InputArrayWrongType"
    assert product(a=None) == product(a_scale=None) == product(w=None) == product(w_scale=None) == product(y=None) == "NullPointer"
    assert product(k=0) == product(n=0) == "InputTensorsWrongShape"
    assert product(rows=1 << 31) == product(n=1 << 31) == product(k=1 << 17) == product(w_stride=1 << 62) == "TooLarge"
    assert product(rows=0, a=None, y=None) == "OK"

    def grouped(groups=2, offsets=p):
        return name(L.zant_b200_qmatmul_grouped(None, p, 2, 8, 0, p, p, groups, 3, 0, p, None, offsets, 0, p, 0))
    assert grouped() == "CudaUnavailable" and grouped(offsets=None) == "NullPointer"
    assert grouped(groups=0) == "InputTensorsWrongShape" and grouped(groups=1025) == "TooLarge"

    def logprobs(dtype=0, x=p, rows=2, vocab=8, stride=0, tokens=p, logprob=p, entropy=p, top=2, ids=p, likely=p):
        return name(L.zant_b200_token_logprobs(None, dtype, x, rows, vocab, stride, tokens, logprob, entropy, top, ids, likely))
    assert logprobs() == logprobs(tokens=None, logprob=None, entropy=None) == logprobs(top=0, ids=None, likely=None) == "CudaUnavailable"
    assert logprobs(tokens=None) == logprobs(logprob=None) == logprobs(ids=None) == logprobs(likely=None) == logprobs(x=None) == "NullPointer"
    assert logprobs(stride=7) == "WrongStride" and logprobs(dtype=2) == "InputArrayWrongType"
    assert logprobs(top=9) == logprobs(top=33, vocab=64) == logprobs(top=-1) == "InvalidInput"
    assert logprobs(rows=1 << 31) == logprobs(vocab=1 << 31, top=0) == "TooLarge"
    assert logprobs(rows=0, x=None) == "OK"


def test_counts_next_to_an_ints_limit(zb):
    """What the loops of the kernels could not step over is refused, a little less is not."""
    L, p = zb.lib(), np.zeros(64, F).__array_interface__["data"][0]
    name = lambda status: L.zant_b200_status_name(C.c_int32(status)).decode()
    for v, want in ((0x7fffffff, "TooLarge"), (0x7fff0001, "TooLarge"), (0x7fff0000, "CudaUnavailable")):
        assert name(L.zant_b200_quantize_rows(None, 0, p, v, 1, 0, None, v, p, 0, p)) == want
        assert name(L.zant_b200_quantize_rows(None, 0, p, 1, v, 0, None, 1, p, 0, p)) == want
        assert name(L.zant_b200_qmatmul_scaled(None, p, v, 1, 0, p, p, 1, 0, p, None, 0, p, 0)) == want
        assert name(L.zant_b200_qmatmul_scaled(None, p, 1, 1, 0, p, p, v, 0, p, None, 0, p, 0)) == want
        assert name(L.zant_b200_token_logprobs(None, 0, p, v, 1, 0, None, None, p, 0, None, None)) == want
        assert name(L.zant_b200_token_logprobs(None, 0, p, 1, v, 0, None, None, p, 0, None, None)) == want


def test_other_operators_refuse_the_new_types(zb):
    L = zb.lib()
    p = np.zeros(64, F).__array_interface__["data"][0]
    sh = (C.c_size_t * 2)(2, 4)
    for dtype in (4, 5):
        assert L.zant_b200_status_name(C.c_int32(L.zant_b200_transpose_onnx(None, C.c_int32(dtype), C.c_void_p(p), sh, C.c_size_t(2), None, C.c_size_t(0), C.c_void_p(p), sh, C.c_size_t(2)))) == b"InputArrayWrongType"
        assert L.zant_b200_status_name(C.c_int32(L.zant_b200_dequantize_linear(None, dtype, p, 8, 1.0, 0, p))) == b"InputArrayWrongType"


def test_results_that_may_not_be_written(zb, nogpu):
    """Read-only arrays (of bytes, of a file mapped for reading) are refused where a result would go."""
    def ro(v):
        v.flags.writeable = False
        return v
    x, a, s, w, ws = np.ones((3, 8), F), np.ones((3, 8), np.int8), np.ones(3, F), np.ones((5, 8), np.int8), np.ones(5, F)
    fixed = np.frombuffer(bytes(24), np.int8).reshape(3, 8)
    refused(zb, "InputArrayWrongType", lambda: nogpu.quantize_rows(x, out=fixed))
    refused(zb, "InputArrayWrongType", lambda: nogpu.quantize_rows(x, out_scale=ro(np.zeros(3, F))))
    refused(zb, "InputArrayWrongType", lambda: nogpu.qmatmul_scaled(a, s, w, ws, out=ro(np.zeros((3, 5), F))))
    refused(zb, "InputArrayWrongType", lambda: nogpu.qmatmul_grouped(a, s, w[None], ws[None], [0, 3], out=ro(np.zeros((3, 5), F))))
    good = [np.zeros(3, F), np.zeros(3, F), np.zeros((3, 2), np.int32), np.zeros((3, 2), F)]
    for i in range(4):
        out = [v.copy() for v in good]
        ro(out[i])
        refused(zb, "InputArrayWrongType", lambda: nogpu.token_logprobs(x, [0, 1, 2], top=2, out=tuple(out)))
    refused(zb, "CudaUnavailable", lambda: nogpu.token_logprobs(ro(x), ro(np.zeros(3, np.int32)), top=2, out=tuple(good)))
