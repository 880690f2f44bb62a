"""Numbers of sinks next to the end of int32 beside windows that a sequence has outgrown: every token is a sink, and every query sees all that is before it."""
import pytest

from test_gpu_kv_attention import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sinks", [2 ** 31 - 129, 2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 32, 2 ** 31 - 31, 2 ** 31 - 16, 2 ** 31 - 15, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("window", [1, 64])
@pytest.mark.parametrize("kind,new,length,dim", [("bf16", 2, 500, 64), ("f32", 3, 300, 256), ("bf16", 150, 500, 128), ("f16", 130, 400, 256)])
def test_every_token_is_a_sink(ctx, zb, kind, new, length, dim, window, sinks):
    check(ctx, zb, [new], [length], 2, 1, dim, 32, kind, window=window, sinks=sinks)


@pytest.mark.parametrize("sinks", [2 ** 31 - 200, 2 ** 31 - 1])
def test_long_contexts(ctx, zb, sinks):
    check(ctx, zb, [1], [17000], 4, 1, 64, 16, "bf16", window=100, sinks=sinks)
